// What the 8-bit row kernels share: eight elements of a row at any alignment, reductions over a
// wave and a workgroup, GELU, and the packing of eight values into bytes.
//
// The 8-bit form: s = max|v| / 127 over the values that share a scale, q = rint(v * (127 / max|v|)),
// so v is held to within s / 2.  Zeros only: s = 0, q = 0.  An infinity or a NaN among them: s = NaN,
// q = 0, so that what is computed from the row is NaN instead of plausible numbers.
#pragma once

#include "common.h"

namespace fmoe {

typedef int32_t i32x4 __attribute__((ext_vector_type(4)));

constexpr int kRowsPitch = 128;  // bytes that a row in 8 bits is padded to
constexpr int kHoldBlock = 128;  // columns of a held activation that share a scale

// ---- eight consecutive elements ---------------------------------------------------------------
// Rows start wherever a tensor's row starts: at any multiple of the element's size.  The vector
// types below carry that alignment, which the device's unaligned access mode serves with the same
// 16-byte instructions (odd row lengths cost a second cache line per access, not scalar loads).
typedef uint32_t u32x4_any __attribute__((ext_vector_type(4), aligned(2)));
typedef uint32_t u32x2_any __attribute__((ext_vector_type(2), aligned(1)));

template <typename T> struct Eight {
  static constexpr int kWords = 2 * ElemInfo<T>::kBytes;  // 32-bit words of eight elements
  using V = Vec<T, 8>;
  using raw_t = typename V::raw_t;

  static __device__ __forceinline__ raw_t zero() {
    raw_t r;
#pragma unroll
    for (int i = 0; i < kWords; ++i) r[i] = 0;
    return r;
  }
  // Elements [col, col + 8) of a row of n: those beyond its end read as zero.
  template <bool NT>
  static __device__ __forceinline__ raw_t load(const T* row, int64_t col, int64_t n) {
    raw_t r = zero();
    if (col + 8 <= n) {
      const u32x4_any* p = reinterpret_cast<const u32x4_any*>(row + col);
      const u32x4 a = NT ? __builtin_nontemporal_load(p) : *p;
      if constexpr (kWords == 4) {
        r = a;
      } else {
        const u32x4 b = NT ? __builtin_nontemporal_load(p + 1) : p[1];
        r = raw_t{a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
      }
    } else if (col < n) {  // one thread of a row at most
      float f[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) f[i] = col + i < n ? ld1(row + col + i) : 0.f;
      r = V::pack(f);
    }
    return r;
  }
  // NT: past the caches, for results that would not stay in them.
  template <bool NT = false>
  static __device__ __forceinline__ void store(T* row, int64_t col, int64_t n, raw_t r) {
    if (col + 8 <= n) {
      u32x4_any* p = reinterpret_cast<u32x4_any*>(row + col);
      const u32x4 a = {r[0], r[1], r[2], r[3]};
      if constexpr (NT) __builtin_nontemporal_store(a, p);
      else *p = a;
      if constexpr (kWords == 8) {
        const u32x4 b = {r[4], r[5], r[6], r[7]};
        if constexpr (NT) __builtin_nontemporal_store(b, p + 1);
        else p[1] = b;
      }
    } else if (col < n) {
      float f[8];
      V::cvt(r, f);
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (col + i < n) st1(row + col + i, f[i]);
    }
  }
};

// ---- reductions -------------------------------------------------------------------------------
template <int CTRL> __device__ __forceinline__ uint32_t dpp(uint32_t v) {
  return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xf, 0xf, true);
}
// All 16 lanes of a DPP row get the row's maximum (sum): rotations by 8, 4, 2 and 1.
__device__ __forceinline__ uint32_t row_max(uint32_t v) {
  v = max(v, dpp<0x128>(v));
  v = max(v, dpp<0x124>(v));
  v = max(v, dpp<0x122>(v));
  return max(v, dpp<0x121>(v));
}
__device__ __forceinline__ float row_sum(float v) {
  v += __uint_as_float(dpp<0x128>(__float_as_uint(v)));
  v += __uint_as_float(dpp<0x124>(__float_as_uint(v)));
  v += __uint_as_float(dpp<0x122>(__float_as_uint(v)));
  return v + __uint_as_float(dpp<0x121>(__float_as_uint(v)));
}
__device__ __forceinline__ uint32_t wave_max(uint32_t v) {
  v = row_max(v);
  v = max(v, (uint32_t)__shfl_xor((int)v, 16));
  return max(v, (uint32_t)__shfl_xor((int)v, 32));
}
__device__ __forceinline__ float wave_sum(float v) {
  v = row_sum(v);
  v += __shfl_xor(v, 16);
  return v + __shfl_xor(v, 32);
}
// Over the THREADS threads of a row: one wave, or the whole workgroup through `lds` (one word per
// wave).  Every thread gets the result; sums are added in wave order, so they repeat bit for bit.
template <int THREADS> __device__ __forceinline__ uint32_t group_max(uint32_t v, uint32_t* lds) {
  v = wave_max(v);
  if constexpr (THREADS > kWave) {
    if ((threadIdx.x & (kWave - 1)) == 0) lds[threadIdx.x / kWave] = v;
    __syncthreads();
    v = lds[0];
#pragma unroll
    for (int i = 1; i < THREADS / kWave; ++i) v = max(v, lds[i]);
  }
  return v;
}
template <int THREADS> __device__ __forceinline__ float group_sum(float v, float* lds) {
  v = wave_sum(v);
  if constexpr (THREADS > kWave) {
    if ((threadIdx.x & (kWave - 1)) == 0) lds[threadIdx.x / kWave] = v;
    __syncthreads();
    v = lds[0];
#pragma unroll
    for (int i = 1; i < THREADS / kWave; ++i) v += lds[i];
  }
  return v;
}

// ---- the 8-bit form ---------------------------------------------------------------------------
// The largest |v| so far.  `maximum` keeps a NaN (fmax would drop it) and is one instruction for two
// values (v_maximum3_f32).  Across lanes the result is compared by its bits: an infinity orders above
// every number and a NaN above the infinities.
__device__ __forceinline__ float larger(float top, float v) {
  return __builtin_elementwise_maximum(top, __builtin_fabsf(v));
}
__device__ __forceinline__ uint32_t abs_bits(float v) { return __float_as_uint(v) & 0x7fffffffu; }

struct Scale8 {
  float scale;  // what a step stands for
  float inv;    // 127 / max
  bool bad;     // an infinity or a NaN among the values
};
__device__ __forceinline__ Scale8 scale8(uint32_t top_bits) {
  const float top = __uint_as_float(top_bits);
  Scale8 s;
  s.bad = top_bits >= 0x7f800000u;
  // the quotient of the largest fp32 number rounds up, and 127 of it are infinite: one step less
  s.scale = s.bad ? __uint_as_float(0x7fc00000u) : fminf(top / 127.0f, 0x1.020406p+121f);
  // Below 2^-118 the scale would be denormal, and a little lower the quotient overflows: such rows
  // are held as zeros.
  const bool zero = top < 0x1p-118f;
  if (zero) s.scale = 0.f;
  s.inv = (s.bad || zero) ? 0.f : 127.0f / top;
  return s;
}
// Eight values as bytes.  v * inv lies in [-127.00002, 127.00002]; adding 1.5 * 2^23 rounds it to
// the nearest whole number (ties to even) and leaves that number's two's complement in the low byte.
__device__ __forceinline__ u32x2 pack8(const float* v, const Scale8& s) {
  uint32_t b[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) b[i] = __float_as_uint(v[i] * s.inv + 12582912.0f);
  u32x2 r;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const uint32_t lo = __builtin_amdgcn_perm(b[4 * i + 1], b[4 * i], 0x0c0c0400u);
    const uint32_t hi = __builtin_amdgcn_perm(b[4 * i + 3], b[4 * i + 2], 0x0c0c0400u);
    r[i] = __builtin_amdgcn_perm(hi, lo, 0x05040100u);
  }
  return s.bad ? u32x2{0u, 0u} : r;
}
__device__ __forceinline__ void unpack8(u32x2 q, float scale, float* v) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int32_t w = (int32_t)q[i / 4];
    v[i] = (float)((w << (24 - 8 * (i % 4))) >> 24) * scale;
  }
}

// ---- GELU ---------------------------------------------------------------------------------------
// gelu(x) = x * Phi(x) with Phi the normal distribution function.  For 16-bit types Phi(x) is
// 1 / (1 + 2^-(x * P(x^2))): the log-odds of Phi are odd and smooth, so P is a polynomial in x^2,
// fitted here by reweighted least squares up to |x| = T; beyond, both stay positive and x * P(x^2)
// rises, so Phi goes to 0 or 1.  With degree 8 and T = 5.5, x * Phi is within 4e-7 of the true value,
// and relatively within 2e-5 down to x = -T; with degree 6 and T = 5 within 3e-6, relatively 2.4e-4:
// a sixteenth of bf16's half step.  13 and 11 instructions and two quarter-rate ones (2^x, 1 / x) an
// element, where erf takes about 50: at 2 bytes an element those bound the kernels instead of HBM
// (49152 x 2048 to 8 bits: 58.5 us with degree 6, 61.5 with 8).  A result of bf16 takes degree 6, one of fp16
// degree 8, and so do rows that go to 8 bits, whatever their type: there an error moves values near a border to
// the next whole number, which shows even beside bf16's rounding (restored rows of a prompt against 64
// bits: 1.61e-3 with degree 6, 1.56e-3 with 8, 1.56e-3 with erf).
// fp32 values take erfc.  Its argument is rounded to within 2^-23 of itself, which the tail amplifies: the
// result's relative error is up to (x^2 + 2) * 2^-23 for a negative x (1e-5 at x = -10, where 1 + erf has no
// bits left), and a few half steps around and above zero.
template <typename T> __device__ __forceinline__ float normal_cdf(float x) {
  if constexpr (ElemInfo<T>::kBytes == 4) {
    return 0.5f * erfcf(-0.70710678118654752f * x);
  } else if constexpr (std::is_same<T, f16_t>::value) {
    const float u = x * x;
    float p = 1.4901355e-12f;
    p = __builtin_fmaf(p, u, -2.3464275e-10f);
    p = __builtin_fmaf(p, u, 1.5883325e-08f);
    p = __builtin_fmaf(p, u, -6.0139405e-07f);
    p = __builtin_fmaf(p, u, 1.3664561e-05f);
    p = __builtin_fmaf(p, u, -1.7102394e-04f);
    p = __builtin_fmaf(p, u, -6.5581713e-05f);
    p = __builtin_fmaf(p, u, 1.0480524e-01f);
    p = __builtin_fmaf(p, u, 2.3022187f);
    return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-(p * x)));
  } else {
    const float u = x * x;
    float p = 2.4839388e-09f;
    p = __builtin_fmaf(p, u, -2.2724015e-07f);
    p = __builtin_fmaf(p, u, 8.1067028e-06f);
    p = __builtin_fmaf(p, u, -1.2739214e-04f);
    p = __builtin_fmaf(p, u, -2.3266282e-04f);
    p = __builtin_fmaf(p, u, 1.0507021e-01f);
    p = __builtin_fmaf(p, u, 2.3020976f);
    return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-(p * x)));
  }
}
// x = -inf would give -inf * 0: the least number stands for it, whose GELU is -0, the limit.  (`maximum`
// keeps a NaN.)
template <typename T> __device__ __forceinline__ float gelu(float x) {
  x = __builtin_elementwise_maximum(x, -3.402823466e38f);
  return x * normal_cdf<T>(x);
}
// The same of a value that goes to 8 bits.
template <typename T> __device__ __forceinline__ float gelu8(float x) {
  return gelu<std::conditional_t<std::is_same<T, bf16_t>::value, f16_t, T>>(x);
}
// d gelu / dx = Phi(x) + x * phi(x), for a finite x (or NaN).
__device__ __forceinline__ float gelu_slope(float x, float cdf) {
  const float e = __builtin_amdgcn_exp2f(-0.72134752f * (x * x));
  return __builtin_fmaf(0.39894228f * x, e, cdf);
}

}  // namespace fmoe
