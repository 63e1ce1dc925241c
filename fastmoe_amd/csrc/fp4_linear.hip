// Every expert's product of 16-bit rows with weights in 4 bits, and weights to 4 bits and back:
//
//   out[r, n] = act(sum_k x[i(r), k] * w[e(r), n, k] + b[e(r), n])
//
// for packed rows r in [off[e], off[e + 1]) of expert e; i(r) = index[r] where the rows are read through an
// index (the dispatch's reverse map), else r; act: nothing, or GELU.
//
// A weight is v * 2^(s - 127): v one of 0, 0.5, 1, 1.5, 2, 3, 4, 6 and their negatives (sign, two bits of exponent, one of
// mantissa), s a byte for 32 neighbouring weights of an output (255: NaN).  That is the form that gfx950 converts two
// of in one instruction, the scale with them, to bf16 or fp16, so the products run on the 16-bit matrix units
// with the rows as they are: bf16 holds such a weight exactly; fp16 does where 2^-23 <= scale <= 2^13, smaller ones are
// rounded to its smallest numbers and larger ones pass its range.  Products are exact and summed in fp32; the result is
// rounded once, to the output's type.
//
// Weights lie with K innermost, two a byte, the earlier one in the low half, padded with zeros to whole pieces of 128; the
// rows end with K.
#include "expert_tiles.h"

#include <cmath>

namespace fmoe {

constexpr int kFp4Block = 32;   // weights that share a scale
constexpr int kFp4Pitch = 128;  // weights of a row are padded to whole pieces of this many

struct Fp4Args {
  const void* x;
  int64_t x_stride;  // elements
  int64_t x_rows;
  const void* index;  // [rows], or null: row r reads row r
  int index_dtype;
  const uint8_t* w;   // [E, N, Kp / 2]
  const uint8_t* s;   // [E, N, Kp / 32]
  const void* bias;   // [E, N], or null
  int bias_dtype;
  int gelu;
  const int64_t* off;  // [E + 1], or null: one expert has every row
  int64_t E, N, K, Kp, rows;
  void* out;
  int64_t out_stride;  // elements
  int groups_n;        // workgroups side by side that cover N
};

typedef float f32x4 __attribute__((ext_vector_type(4)));

// Eight 16-bit values of a matrix unit's operand, and its products.
template <typename T> struct Operand;
template <> struct Operand<bf16_t> {
  typedef __bf16 type __attribute__((ext_vector_type(8)));
  static __device__ __forceinline__ f32x4 mfma16(u32x4 a, u32x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(type, a), __builtin_bit_cast(type, b), c, 0, 0, 0);
  }
  // Eight weights with their scale, of which only the exponent's bits are read.
  static __device__ __forceinline__ u32x4 weights(uint32_t w, float s) {
    return u32x4{__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s, 0)),
                 __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s, 1)),
                 __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s, 2)),
                 __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s, 3))};
  }
};
template <> struct Operand<f16_t> {
  typedef _Float16 type __attribute__((ext_vector_type(8)));
  static __device__ __forceinline__ f32x4 mfma16(u32x4 a, u32x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(type, a), __builtin_bit_cast(type, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ u32x4 weights(uint32_t w, float s) {
    return u32x4{__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, s, 0)),
                 __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, s, 1)),
                 __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, s, 2)),
                 __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, s, 3))};
  }
};

// The scale of byte `at` of four.
__device__ __forceinline__ float scale_of(uint32_t four, int at) {
  return __uint_as_float((four >> (8 * at) & 0xff) << 23);
}

// Four neighbouring columns of one output row, of which those from `n` to N are there.
template <typename TO>
__device__ __forceinline__ void store4(const Fp4Args& a, const Tile& t, int64_t r, int64_t n, f32x4 acc) {
  if (n >= a.N) return;
  TO* p = static_cast<TO*>(a.out) + r * a.out_stride + n;
  const int left = (int)min((int64_t)4, a.N - n);
  float f[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    f[i] = acc[i];
    if (a.bias && i < left) f[i] += load_weight(a.bias, a.bias_dtype, t.expert * a.N + n + i);
    if (a.gelu) f[i] = gelu<TO>(f[i]);
  }
  apart<TO>(f);
  if (left == 4) {
    if constexpr (ElemInfo<TO>::kBytes == 4) *reinterpret_cast<u32x4_any*>(p) = Vec<TO, 4>::pack(f);
    else *reinterpret_cast<u32x2_any*>(p) = Vec<TO, 4>::pack(f);
  } else {
    for (int i = 0; i < left; ++i) st1(p + i, f[i]);
  }
}

// Few rows: 16 rows by 16 columns in a workgroup, whose eight waves take pieces of 128 of K in turn, straight from memory to
// the matrix units' registers, and add their parts in LDS in one order.
constexpr int kFp4Waves = 8;
template <typename TX, typename TO> __global__ __launch_bounds__(kFp4Waves * kWave) void k_fp4_few(Fp4Args a) {
  __shared__ f32x4 part[kFp4Waves][kWave];
  Tile t;
  int group;
  if (!place<16>(a, &t, &group)) return;
  const int64_t n0 = (int64_t)group * 16;
  if (t.expert == a.E) {
    zero_rows<TO>(a, t, n0, 16);
    return;
  }
  const int lane = threadIdx.x & (kWave - 1), wave = uniform(threadIdx.x / kWave);
  const int l16 = lane & 15, quad = lane >> 4;
  // lane l has row (of x) or column (of the weights) l % 16 and 32 of a piece's K from 32 * (l / 16) on; the
  // order of K is the same for both, so eight of them at a time are as good as any
  const int64_t row = source_row(a, t.row + min(l16, t.count - 1));
  const bool live = l16 < t.count && row >= 0;
  const TX* xp = static_cast<const TX*>(a.x) + max(row, (int64_t)0) * a.x_stride;
  const int64_t col = t.expert * a.N + min(n0 + l16, a.N - 1);
  const uint8_t* wp = a.w + col * (a.Kp / 2) + quad * 16;
  const uint8_t* sp = a.s + col * (a.Kp / kFp4Block);
  f32x4 acc = {0.f, 0.f, 0.f, 0.f};
  for (int64_t k = wave * 128; k < a.Kp; k += kFp4Waves * 128) {
    const u32x4 w = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(wp + k / 2));
    const float scale = scale_of(*reinterpret_cast<const uint32_t*>(sp + k / kFp4Block), quad);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int64_t at = k + quad * 32 + j * 8;
      const u32x4 x = live ? Eight<TX>::template load<false>(xp, at, a.K) : Eight<TX>::zero();
      acc = Operand<TX>::mfma16(Operand<TX>::weights(w[j], scale), x, acc);
    }
  }
  part[wave][lane] = acc;
  __syncthreads();
  if (wave != 0 || l16 >= t.count) return;
#pragma unroll
  for (int v = 1; v < kFp4Waves; ++v) acc += part[v][lane];
  // lane l of a 16 x 16 result has row l % 16 and columns 4 * (l / 16) + 0..3
  store4<TO>(a, t, t.row + l16, n0 + quad * 4, acc);
}

// ---- weights to 4 bits and back ---------------------------------------------------------------------
// A thread takes the 32 weights of a scale: the smallest power of two with which none of them passes 6.
template <typename T> __global__ __launch_bounds__(kGroup) void k_to_fp4(const T* x, int64_t stride, int64_t rows,
                                                                         int64_t cols, int64_t blocks, uint8_t* q,
                                                                         uint8_t* s) {
  const int64_t i = (int64_t)blockIdx.x * kGroup + threadIdx.x;
  if (i >= rows * blocks) return;
  const int64_t row = i / blocks, col = i % blocks * kFp4Block;
  float f[32];
  float top = 0.f;
#pragma unroll
  for (int v = 0; v < 4; ++v) {
    Eight<T>::V::cvt(Eight<T>::template load<false>(x + row * stride, col + v * 8, cols), f + v * 8);
#pragma unroll
    for (int j = 0; j < 8; ++j) top = larger(top, f[v * 8 + j]);
  }
  u32x4 out = {0, 0, 0, 0};
  int exponent = 255;  // an infinity or a NaN among them: NaN, so that what is computed from them is NaN
  if (abs_bits(top) < 0x7f800000u) {
    int e;
    const float m = __builtin_frexpf(top, &e);  // top = m 2^e, 0.5 <= m < 1; 6 = 0.75 * 2^3
    exponent = top == 0.f ? 127 : max(e - 3 + (m > 0.75f ? 1 : 0), -127) + 127;
    const float scale = __builtin_ldexpf(1.f, exponent - 127);
#pragma unroll
    for (int v = 0; v < 4; ++v) {
      uint32_t w = 0;  // nearest, ties to even
      w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, f[8 * v], f[8 * v + 1], scale, 0);
      w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, f[8 * v + 2], f[8 * v + 3], scale, 1);
      w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, f[8 * v + 4], f[8 * v + 5], scale, 2);
      w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, f[8 * v + 6], f[8 * v + 7], scale, 3);
      out[v] = w;
    }
  }
  *reinterpret_cast<u32x4*>(q + i * (kFp4Block / 2)) = out;
  s[i] = (uint8_t)exponent;
}

template <typename T> __global__ __launch_bounds__(kGroup) void k_from_fp4(const uint8_t* q, const uint8_t* s,
                                                                           int64_t rows, int64_t cols, int64_t blocks,
                                                                           T* out) {
  const int64_t i = (int64_t)blockIdx.x * kGroup + threadIdx.x;
  if (i >= rows * blocks) return;
  const int64_t row = i / blocks, col = i % blocks * kFp4Block;
  if (col >= cols) return;
  const u32x4 w = *reinterpret_cast<const u32x4*>(q + i * (kFp4Block / 2));
  const float scale = __uint_as_float((uint32_t)s[i] << 23);
#pragma unroll
  for (int v = 0; v < 4; ++v) {
    typename Eight<T>::raw_t r;
    if constexpr (ElemInfo<T>::kBytes == 4) {
      const auto put = [&](auto p, int at) {
        r[at] = __float_as_uint(p[0]);
        r[at + 1] = __float_as_uint(p[1]);
      };
      put(__builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[v], scale, 0), 0);
      put(__builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[v], scale, 1), 2);
      put(__builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[v], scale, 2), 4);
      put(__builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[v], scale, 3), 6);
    } else {
      r = Operand<T>::weights(w[v], scale);
    }
    Eight<T>::store(out + row * cols, col + v * 8, cols, r);
  }
}

}  // namespace fmoe

using namespace fmoe;

namespace {

template <typename TX, typename TO> int launch_few(const char* who, Fp4Args a, hipStream_t s) {
  const int64_t groups = grid_of(who, &a, 16, 16, kFp4Waves * kWave);
  if (groups < 0) return FMOE_ERANGE;
  hipLaunchKernelGGL((k_fp4_few<TX, TO>), dim3((unsigned)groups), dim3(kFp4Waves * kWave), 0, s, a);
  return fmoe_host::check_launch(who);
}

template <typename TX, typename TO> int launch_linear(const char* who, const Fp4Args& a, hipStream_t s) {
  return launch_few<TX, TO>(who, a, s);
}

int check_fp4(const char* who, int64_t rows, int64_t cols, const void* q, const void* s) {
  FMOE_REQUIRE(rows >= 0 && cols >= 1, "%s: bad sizes rows=%lld columns=%lld", who, (long long)rows, (long long)cols);
  if (rows >= (int64_t(1) << 31) || cols > (int64_t(1) << 24) ||
      rows * (fmoe_host::round_up(cols, kFp4Pitch) / kFp4Block) > (int64_t(1) << 31)) {
    fmoe_host::set_error("%s: rows=%lld columns=%lld too large", who, (long long)rows, (long long)cols);
    return FMOE_ERANGE;
  }
  FMOE_REQUIRE(rows == 0 || (q && s), "%s: null device pointer", who);
  FMOE_REQUIRE(reinterpret_cast<uintptr_t>(q) % 16 == 0, "%s: 4-bit weights must start at a multiple of 16 bytes", who);
  return FMOE_OK;
}

}  // namespace

extern "C" int fmoe_quantize_fp4(const void* d_x, int64_t x_row_stride, int64_t rows, int64_t cols, int dtype,
                                 void* d_q, void* d_scales, void* stream) {
  fmoe_host::clear_error();
  const char* who = "fmoe_quantize_fp4";
  FMOE_REQUIRE(fmoe_host::is_float_dtype(dtype), "%s: bad dtype %d", who, dtype);
  if (int rc = check_fp4(who, rows, cols, d_q, d_scales)) return rc;
  FMOE_REQUIRE(x_row_stride >= 0 && (rows == 0 || d_x), "%s: null device pointer or negative row stride", who);
  if (rows == 0) return FMOE_OK;
  const int64_t blocks = fmoe_host::round_up(cols, kFp4Pitch) / kFp4Block;
  const dim3 grid((unsigned)((rows * blocks + kGroup - 1) / kGroup));
  hipStream_t s = static_cast<hipStream_t>(stream);
  auto go = [&](auto t) {
    using T = decltype(t);
    hipLaunchKernelGGL((k_to_fp4<T>), grid, dim3(kGroup), 0, s, static_cast<const T*>(d_x), x_row_stride, rows, cols,
                       blocks, static_cast<uint8_t*>(d_q), static_cast<uint8_t*>(d_scales));
  };
  if (dtype == FMOE_F32) go(float{});
  else if (dtype == FMOE_BF16) go(bf16_t{});
  else go(f16_t{});
  return fmoe_host::check_launch(who);
}

extern "C" int fmoe_restore_fp4(const void* d_q, const void* d_scales, int64_t rows, int64_t cols, void* d_out,
                                int dtype, void* stream) {
  fmoe_host::clear_error();
  const char* who = "fmoe_restore_fp4";
  FMOE_REQUIRE(fmoe_host::is_float_dtype(dtype), "%s: bad dtype %d", who, dtype);
  if (int rc = check_fp4(who, rows, cols, d_q, d_scales)) return rc;
  FMOE_REQUIRE(rows == 0 || d_out, "%s: null device pointer", who);
  if (rows == 0) return FMOE_OK;
  const int64_t blocks = fmoe_host::round_up(cols, kFp4Pitch) / kFp4Block;
  const dim3 grid((unsigned)((rows * blocks + kGroup - 1) / kGroup));
  hipStream_t s = static_cast<hipStream_t>(stream);
  auto go = [&](auto t) {
    using T = decltype(t);
    hipLaunchKernelGGL((k_from_fp4<T>), grid, dim3(kGroup), 0, s, static_cast<const uint8_t*>(d_q),
                       static_cast<const uint8_t*>(d_scales), rows, cols, blocks, static_cast<T*>(d_out));
  };
  if (dtype == FMOE_F32) go(float{});
  else if (dtype == FMOE_BF16) go(bf16_t{});
  else go(f16_t{});
  return fmoe_host::check_launch(who);
}

extern "C" int fmoe_fp4_linear(const void* d_x, int64_t x_row_stride, int64_t x_rows, int x_dtype,
                               const void* d_index, int index_dtype, const void* d_w, const void* d_w_scales,
                               const void* d_bias, int bias_dtype, int activation, const int64_t* d_offsets,
                               int64_t num_experts, int64_t N, int64_t K, int64_t rows, void* d_out,
                               int64_t out_row_stride, int out_dtype, void* stream) {
  fmoe_host::clear_error();
  const char* who = "fmoe_fp4_linear";
  FMOE_REQUIRE(rows >= 0 && x_rows >= 0 && N >= 1 && K >= 1 && num_experts >= 1,
               "%s: bad sizes rows=%lld x_rows=%lld N=%lld K=%lld E=%lld", who, (long long)rows,
               (long long)x_rows, (long long)N, (long long)K, (long long)num_experts);
  FMOE_REQUIRE(x_dtype == FMOE_BF16 || x_dtype == FMOE_F16, "%s: rows must be bf16 or fp16, got dtype %d", who, x_dtype);
  FMOE_REQUIRE(fmoe_host::is_float_dtype(out_dtype), "%s: bad output dtype %d", who, out_dtype);
  FMOE_REQUIRE(!d_index || fmoe_host::is_index_dtype(index_dtype), "%s: bad index dtype %d", who, index_dtype);
  FMOE_REQUIRE(!d_bias || fmoe_host::is_float_dtype(bias_dtype), "%s: bad bias dtype %d", who, bias_dtype);
  FMOE_REQUIRE(activation == FMOE_ACT_NONE || activation == FMOE_ACT_GELU, "%s: bad activation %d", who, activation);
  FMOE_REQUIRE(d_offsets || num_experts == 1, "%s: several experts need row offsets", who);
  FMOE_REQUIRE(out_row_stride >= N, "%s: out row stride %lld is below N=%lld", who, (long long)out_row_stride,
               (long long)N);
  FMOE_REQUIRE(x_row_stride >= 0, "%s: negative row stride", who);
  FMOE_REQUIRE(reinterpret_cast<uintptr_t>(d_w) % 16 == 0 && reinterpret_cast<uintptr_t>(d_w_scales) % 4 == 0,
               "%s: weights must start at a multiple of 16 bytes, their scales of 4", who);
  if (K > (int64_t(1) << 17) || N > (int64_t(1) << 24) || num_experts > (int64_t(1) << 16) ||
      rows >= (int64_t(1) << 31) || x_rows >= (int64_t(1) << 31)) {
    fmoe_host::set_error("%s: rows=%lld x_rows=%lld N=%lld K=%lld E=%lld too large", who, (long long)rows,
                         (long long)x_rows, (long long)N, (long long)K, (long long)num_experts);
    return FMOE_ERANGE;
  }
  if (rows == 0) return FMOE_OK;
  FMOE_REQUIRE(x_rows >= 1, "%s: rows to write, and none to read", who);
  FMOE_REQUIRE(d_x && d_w && d_w_scales && d_out, "%s: null device pointer", who);
  const Fp4Args a{d_x, x_row_stride, x_rows, d_index, index_dtype, static_cast<const uint8_t*>(d_w),
                  static_cast<const uint8_t*>(d_w_scales), d_bias, bias_dtype, activation == FMOE_ACT_GELU, d_offsets,
                  num_experts, N, K, fmoe_host::round_up(K, kFp4Pitch), rows, d_out, out_row_stride, 0};
  hipStream_t s = static_cast<hipStream_t>(stream);
  auto from = [&](auto tx) {
    using TX = decltype(tx);
    if (out_dtype == FMOE_F32) return launch_linear<TX, float>(who, a, s);
    if (out_dtype == FMOE_BF16) return launch_linear<TX, bf16_t>(who, a, s);
    return launch_linear<TX, f16_t>(who, a, s);
  };
  return x_dtype == FMOE_BF16 ? from(bf16_t{}) : from(f16_t{});
}
