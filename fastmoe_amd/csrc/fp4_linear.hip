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
// with the rows as they are: bf16 holds such a weight exactly where fp32 does; fp16 does where 2^-23 <= scale <= 2^13, smaller ones are
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
  int out_dtype;
  int groups_n;        // workgroups side by side that cover N
};

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

// Eight 16-bit values of a matrix unit's operand, and its products.
template <typename T> struct Operand;
template <> struct Operand<bf16_t> {
  typedef __bf16 type __attribute__((ext_vector_type(8)));
  static __device__ __forceinline__ f32x4 mfma16(u32x4 a, u32x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(type, a), __builtin_bit_cast(type, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ f32x16 mfma32(u32x4 a, u32x4 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(type, a), __builtin_bit_cast(type, b), c, 0, 0, 0);
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
  static __device__ __forceinline__ f32x16 mfma32(u32x4 a, u32x4 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(type, a), __builtin_bit_cast(type, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ u32x4 weights(uint32_t w, float s) {
    return u32x4{__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, s, 0)),
                 __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, s, 1)),
                 __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, s, 2)),
                 __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, s, 3))};
  }
};

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

// f(a value of the output's type)
template <typename F> __device__ __forceinline__ void by_output(const Fp4Args& a, F&& f) {
  if (a.out_dtype == FMOE_F32) f(float{});
  else if (a.out_dtype == FMOE_BF16) f(bf16_t{});
  else f(f16_t{});
}

// Few rows: up to 16, by 16 columns for each of a workgroup's eight waves, or for each KS of them, which then take pieces
// of 256 of K in turn and add their parts in LDS in one order.  A wave brings its own weights through a ring of three buffers in
// LDS, eight lanes for the 128 bytes of a column's piece: whole lines.  (Straight to the matrix units' registers, where
// neighbouring lanes have different columns, they came at 3.1 TB/s, whatever the waves and pieces in flight.)  256 experts'
// [2048, 2048] (570 MB) at 4 rows each take 122 us: 4.7 TB/s.
// The rows lie in LDS, as much of K at a time as fits.  No wave waits for another but where the next part of the rows comes.
constexpr int kFewWaves = 8;
// Bytes of LDS for rows: at least a round of all waves' pieces of 16 rows; where K is split over one or two, two workgroups
// share a CU's.
template <int KS> constexpr int few_bytes() { return KS > 2 ? 16 * 256 * KS * 2 : 24576; }
template <typename TX, int KS> __global__ __launch_bounds__(kFewWaves * kWave) void k_fp4_few(Fp4Args a) {
  constexpr int BN = 16 * (kFewWaves / KS), kFewBytes = few_bytes<KS>();
  constexpr int kCodes = 16 * 128, kPiece = kCodes + 16 * 8, kLoads = 3;  // codes, then scales, of a wave
  // 16 bytes more for each row: the rows that a read's lanes touch together start in different banks
  __shared__ __attribute__((aligned(16))) uint8_t lds[kFewBytes + 16 * 16];
  // separate objects: the compiler then sees that reads of one need not wait for the loads in flight to the others
  __shared__ __attribute__((aligned(1024))) uint8_t ring0[kFewWaves][kPiece];
  __shared__ __attribute__((aligned(1024))) uint8_t ring1[kFewWaves][kPiece];
  __shared__ __attribute__((aligned(1024))) uint8_t ring2[kFewWaves][kPiece];
  static_assert(KS == 1 || kFewWaves * kWave * 16 <= kFewBytes, "the parts fit where the rows were");
  static_assert(16 * 256 * KS * 2 <= kFewBytes, "a round of 16 rows fits");
  Tile t;
  int group;
  if (!place<16>(a, &t, &group)) return;
  const int64_t n0 = (int64_t)group * BN;
  if (t.expert == a.E) {
    by_output(a, [&](auto to) { zero_rows<decltype(to)>(a, t, n0, BN); });
    return;
  }
  const int lane = threadIdx.x & (kWave - 1), wave = uniform(threadIdx.x / kWave);
  const int l16 = lane & 15, quad = lane >> 4, part = wave % KS;
  const int64_t col0 = n0 + wave / KS * 16;
  auto column = [&](int c) { return t.expert * a.N + min(col0 + c, a.N - 1); };
  const uint8_t* const wp[2] = {a.w + column(lane / 8) * (a.Kp / 2), a.w + column(8 + lane / 8) * (a.Kp / 2)};
  const uint8_t* const sp = a.s + column(lane / 2 % 16) * (a.Kp / kFp4Block);
  const int pieces = (int)((a.Kp + 255) / 256), mine = pieces > part ? (pieces - part + KS - 1) / KS : 0;
  const int beyond = (int)(a.Kp / 64) - quad;  // in 64s of K, where a column ends for this lane
  // Piece j of this wave's.  What lies beyond a column's end is read as its last chunk once more, and meets rows of zeros; its
  // scale is taken as the smallest: another's might make an infinity of these codes.
  auto ask = [&](uint8_t (*ring)[kPiece], int j) __attribute__((always_inline)) {
    const int64_t p = (int64_t)j * KS + part;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int chunk = lane % 8 ^ swizzle<128>(i * 8 + lane / 8);
      load_piece<kCPol>(wp[i] + min(p * 8 + chunk, a.Kp / 32 - 1) * 16, ring[wave] + i * 1024);
    }
    if (lane < 32)
      __builtin_amdgcn_global_load_lds(reinterpret_cast<const FMOE_GLOBAL uint32_t*>(reinterpret_cast<uintptr_t>(
                                           sp + min(p * 2 + lane % 2, a.Kp / 128 - 1) * 4)),
                                       (FMOE_LDS uint32_t*)(ring[wave] + kCodes), 4, 0, kCPolCached);
  };
  if (mine > 0) ask(ring0, 0);
  if (mine > 1) ask(ring1, 1);
  // columns of the rows that LDS holds: whole rounds of the waves' pieces
  const int round = 256 * KS;
  const int held = kFewBytes / 2 / t.count / round * round, pitch = held * 2 + 16;
  auto stage = [&](int64_t from) __attribute__((always_inline)) {
    const int width = (int)min((int64_t)held, pieces * (int64_t)256 - from) / 8;  // 16-byte chunks of a row
    for (int i = threadIdx.x; i < t.count * width; i += kFewWaves * kWave) {
      const int r = i / width, c = i % width;
      const int64_t row = source_row(a, t.row + r);
      const u32x4 v = row < 0 ? Eight<TX>::zero()
                              : Eight<TX>::template load<false>(static_cast<const TX*>(a.x) + row * a.x_stride, from + c * 8, a.K);
      *reinterpret_cast<u32x4*>(lds + r * pitch + c * 16) = v;
    }
  };
  f32x4 acc = {0.f, 0.f, 0.f, 0.f};
  // lane l has row (of x) or column (of the weights) l % 16 and 64 of a piece's K from 64 * (l / 16) on; the
  // order of K is the same for both, so eight of them at a time are as good as any
  const uint8_t* xl = lds + min(l16, t.count - 1) * pitch + quad * 128;
  const int rounds = held / round;         // pieces of this wave in LDS at a time
  const int all = (pieces + KS - 1) / KS;  // the same for every wave: they meet at the barriers
  stage(0);
  __syncthreads();
  int base = 0;  // this wave's first piece in LDS
  auto step = [&](uint8_t (*old)[kPiece], const uint8_t (*cur)[kPiece], int i) __attribute__((always_inline)) {
    if (i - base == rounds) {
      __syncthreads();
      stage((int64_t)i * round);
      __syncthreads();
      base = i;
    }
    if (i >= mine) return;
    if (i + 1 < mine) wait_loads<kLoads>();
    else wait_loads<0>();
    u32x4 w[2];
#pragma unroll
    for (int h = 0; h < 2; ++h)
      w[h] = *reinterpret_cast<const u32x4*>(cur[wave] + l16 * 128 + ((quad * 2 + h) ^ swizzle<128>(l16)) * 16);
    uint32_t e = *reinterpret_cast<const uint16_t*>(cur[wave] + kCodes + l16 * 8 + quad * 2);
    if ((i * KS + part) * 4 >= beyond) e = 0;
    if (i + 2 < mine) ask(old, i + 2);
    const uint8_t* xs = xl + ((i - base) * KS + part) * 512;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const float scale = __uint_as_float((h ? e >> 8 : e & 0xff) << 23);
#pragma unroll
      for (int k = 0; k < 4; ++k)
        acc = Operand<TX>::mfma16(Operand<TX>::weights(w[h][k], scale), *reinterpret_cast<const u32x4*>(xs + h * 64 + k * 16), acc);
    }
  };
  for (int i = 0; i < all; i += 3) {
    step(ring2, ring0, i);
    if (i + 1 < all) step(ring0, ring1, i + 1);
    if (i + 2 < all) step(ring1, ring2, i + 2);
  }
  if constexpr (KS > 1) {
    __syncthreads();
    f32x4(*parts)[kWave] = reinterpret_cast<f32x4(*)[kWave]>(lds);
    parts[wave][lane] = acc;
    __syncthreads();
    if (part != 0) return;
#pragma unroll
    for (int v = 1; v < KS; ++v) acc += parts[wave + v][lane];
  }
  if (l16 >= t.count) return;
  // lane l of a 16 x 16 result has row l % 16 and columns 4 * (l / 16) + 0..3
  by_output(a, [&](auto to) { store4<decltype(to)>(a, t, t.row + l16, col0 + quad * 4, acc); });
}

// Eight 16-bit values without the first n, zeros behind them: where eight lie across a row's end, its last eight are read,
// and moved.  (Read one by one they cost 1501 x 3 rows of 13 experts' [1003, 1001] 3 us of 27.)
__device__ __forceinline__ u32x4 without(u32x4 v, int n) {
  if (n & 1)
    v = u32x4{__builtin_amdgcn_alignbit(v[1], v[0], 16), __builtin_amdgcn_alignbit(v[2], v[1], 16),
              __builtin_amdgcn_alignbit(v[3], v[2], 16), v[3] >> 16};
  if (n & 2) v = u32x4{v[1], v[2], v[3], 0};
  if (n & 4) v = u32x4{v[2], v[3], 0, 0};
  if (n >= 8) v = u32x4{0, 0, 0, 0};
  return v;
}

// TM * 32 rows by 4 * WN * 32 columns of one expert in a workgroup of four waves.  Each wave has every row and its own
// 32 WN columns, so each weight is converted once and a converted one serves all rows.
//
// The rows go in pieces of 64 of K through a ring of three buffers in LDS, which the loads write directly where rows start at
// multiples of 16 bytes and K has whole pieces (DIRECT); else through registers, zeros beyond K.  A wave brings its own
// weights 256 of K at a time, eight lanes for a column's 128 bytes (whole lines: with 32 bytes of a column at a time each line came
// twice, and lines that pass the caches four times), into a buffer of its own, takes all of its codes from there
// into registers, and asks for the next 256 at once: they are on their way while these are multiplied.
//
// In LDS a row's piece and a column's codes are 128 bytes each, their 16-byte chunk c at position c ^ swizzle: what a read's
// lanes touch together then lies in different banks.  Lane l of a matrix unit's operand has row (column) l % 32, and of
// a piece's K the half l / 32: four steps of 8, a chunk of codes for all four.
//
// Many rows are bound by the matrix units at the clock that they leave: 49152 rows of 64 experts' [2048, 4096] in 715 us are 1.15
// PFLOP/s, 63 % of their cycles at 1.95 GHz (a large product of the library's: 1.38).
//
// Weights that one tile of rows reads pass the caches; where more of an expert's tiles read them (AGAIN), they stay: at 128 experts'
// [2048, 7168] 128 rows each take 574 us instead of 607, 768 rows 2460 instead of 2690, but 64 rows 323 instead of 308.
template <typename TX, int TM, int WN, bool DIRECT, bool AGAIN>
__global__ __launch_bounds__(4 * kWave, 2) void k_fp4_tile(Fp4Args a) {
  constexpr int W = 4, BM = TM * 32, BN = W * WN * 32;
  constexpr int kX = BM * 128, kCodes = WN * 32 * 128, kW = WN * 5;  // loads of a wave for 256 of K of its columns
  // separate objects: the compiler then sees that reads of one need not wait for the loads in flight to the others
  __shared__ __attribute__((aligned(1024))) uint8_t rows0[kX];
  __shared__ __attribute__((aligned(1024))) uint8_t rows1[kX];
  __shared__ __attribute__((aligned(1024))) uint8_t rows2[kX];
  __shared__ __attribute__((aligned(1024))) uint8_t weights[W][kCodes + WN * 32 * 8];  // codes, then scales
  __shared__ float col_bias[BN];
  __shared__ uint8_t row_live[BM];
  Tile t;
  int group;
  if (!place<BM>(a, &t, &group)) return;
  const int64_t n0 = (int64_t)group * BN;
  if (t.expert == a.E) {
    by_output(a, [&](auto to) { zero_rows<decltype(to)>(a, t, n0, BN); });
    return;
  }
  const int lane = threadIdx.x & (kWave - 1), wave = uniform(threadIdx.x / kWave);
  const int l32 = lane & 31, half = lane >> 5;
  const int w0 = wave * WN * 32;  // this wave's columns
  // Its columns' codes and scales through descriptors that end with the last column: what lies beyond reads as zero.  A load's
  // whole place is in its vector offset: a scalar one has no part in the range check.
  const int here = (int)max(min((int64_t)WN * 32, a.N - n0 - w0), (int64_t)0);
  const int64_t first = t.expert * a.N + min(n0 + w0, a.N - 1);
  const int code_pitch = (int)(a.Kp / 2), scale_pitch = (int)(a.Kp / kFp4Block);
  const rsrc_t codes_at = make_rsrc(a.w + first * code_pitch, (uint32_t)here * code_pitch);
  const rsrc_t scales_at = make_rsrc(a.s + first * scale_pitch, (uint32_t)here * scale_pitch);
  const int code_from = lane / 8 * code_pitch, scale_from = lane / 2 * scale_pitch + lane % 2 * 4;
  auto load_w = [&](int s, int i) __attribute__((always_inline)) {  // load i of 256 of K
    if (i < 4 * WN) {
      const int chunk = (lane % 8) ^ swizzle<128>(i * 8 + lane / 8);
      __builtin_amdgcn_raw_ptr_buffer_load_lds(codes_at, (FMOE_LDS void*)(weights[wave] + i * 1024), 16,
                                               code_from + chunk * 16 + (i * 8 * code_pitch + s * 128), 0, 0,
                                               AGAIN ? kCPolCached : kCPol);
    } else {
      const int n = i - 4 * WN;
      __builtin_amdgcn_raw_ptr_buffer_load_lds(scales_at, (FMOE_LDS void*)(weights[wave] + kCodes + n * 256), 4,
                                               scale_from + (n * 32 * scale_pitch + s * 8), 0, 0, kCPolCached);
    }
  };
#pragma unroll
  for (int i = 0; i < kW; ++i) load_w(0, i);  // before the rows' places are known
  const TX* xp[TM];
  int xc[TM];  // the column that the lane reads of a piece
#pragma unroll
  for (int m = 0; m < TM; ++m) {
    const int r = m * 32 + wave * 8 + lane / 8;
    xp[m] = static_cast<const TX*>(a.x) + max(source_row(a, t.row + min(r, t.count - 1)), (int64_t)0) * a.x_stride;
    xc[m] = (lane % 8 ^ swizzle<128>(r)) * 8;
    if constexpr (DIRECT) xp[m] += xc[m];
  }
  for (int c = threadIdx.x; c < BN; c += W * kWave)
    col_bias[c] = a.bias ? load_weight(a.bias, a.bias_dtype, t.expert * a.N + min(n0 + c, a.N - 1)) : 0.f;
  for (int r = threadIdx.x; r < BM; r += W * kWave) row_live[r] = source_row(a, t.row + min(r, t.count - 1)) >= 0;
  const int pieces = (int)((a.K + 63) / 64), supers = (pieces + 3) / 4;
  auto load_x = [&](uint8_t* s, int piece, int m) __attribute__((always_inline)) {
    load_piece<kCPolCached>(reinterpret_cast<const uint8_t*>(xp[m] + (int64_t)piece * 64), s + (m * 4 + wave) * 1024);
  };
  u32x4 xr[DIRECT ? 1 : TM];  // the rows' part of a piece on its way
  auto fetch = [&](int piece) __attribute__((always_inline)) {
    if constexpr (!DIRECT)
#pragma unroll
      for (int m = 0; m < TM; ++m) {
        const int64_t col = (int64_t)piece * 64 + xc[m];
        if (a.K >= 8) xr[m] = *reinterpret_cast<const u32x4_any*>(xp[m] + min(col, a.K - 8));
        else xr[m] = Eight<TX>::template load<false>(xp[m], col, a.K);
      }
  };
  auto put = [&](uint8_t* s, int piece) __attribute__((always_inline)) {
    if constexpr (!DIRECT)
#pragma unroll
      for (int m = 0; m < TM; ++m) {
        const int64_t col = (int64_t)piece * 64 + xc[m];
        u32x4 v = xr[m];
        if (a.K >= 8 && (int64_t)piece * 64 + 64 > a.K) v = without(v, (int)(col - min(col, a.K - 8)));
        *reinterpret_cast<u32x4*>(s + (m * 4 + wave) * 1024 + lane * 16) = v;
      }
  };
  f32x16 acc[WN][TM];
#pragma unroll
  for (int n = 0; n < WN; ++n)
#pragma unroll
    for (int m = 0; m < TM; ++m)
#pragma unroll
      for (int i = 0; i < 16; ++i) acc[n][m][i] = 0.f;
  u32x4 xv[2][TM], wv[2][WN];  // operands of this and the next step
  u32x4 codes[WN][4];          // of 256 of K
  uint32_t scales[WN][2];
  auto read_x = [&](const uint8_t* s, int k, int to, int m) __attribute__((always_inline)) {
    xv[to][m] = *reinterpret_cast<const u32x4*>(s + (m * 32 + l32) * 128 + ((half * 4 + k) ^ swizzle<128>(l32)) * 16);
  };
  auto read_w = [&] __attribute__((always_inline)) {
#pragma unroll
    for (int n = 0; n < WN; ++n) {
      const u32x2 s = *reinterpret_cast<const u32x2*>(weights[wave] + kCodes + (n * 32 + l32) * 8);
      scales[n][0] = s[0] >> (8 * half);
      scales[n][1] = s[1] >> (8 * half);
    }
#pragma unroll
    for (int c = 0; c < 4; ++c)
#pragma unroll
      for (int n = 0; n < WN; ++n)
        codes[n][c] = *reinterpret_cast<const u32x4*>(weights[wave] + (n * 32 + l32) * 128 + ((2 * c + half) ^ swizzle<128>(l32)) * 16);
  };
  auto convert = [&](int c, int k, int to) __attribute__((always_inline)) {
#pragma unroll
    for (int n = 0; n < WN; ++n)
      wv[to][n] = Operand<TX>::weights(codes[n][c][k], __uint_as_float((scales[n][c / 2] >> (16 * (c % 2)) & 0xff) << 23));
  };
  // Step i multiplies piece i in buffer `cur`, the part c of 256 of K, by `live` tiles of 32 rows.  Before its last quarter each
  // wave has read all of the piece and waits until its loads of piece i + 1 have arrived; behind the barrier that
  // holds for every wave, so `next` is read, and `cur` is free.  Piece i + 2 is loaded into `old`.
  auto step = [&](auto live, auto part, uint8_t* old, uint8_t* cur, const uint8_t* next, int i)
                  __attribute__((always_inline)) {
    constexpr int kLive = decltype(live)::value, c = decltype(part)::value, kParts = kLive * WN;
    constexpr int kRows = DIRECT ? kLive : 0;  // loads of a wave a piece
    const bool more_x = i + 2 < pieces, more_w = c < 2 && i / 4 + 1 < supers;
    if (more_x) put(old, i + 2);  // what was fetched in the last step
    if (i + 3 < pieces) fetch(i + 3);
    if (c == 0 && more_w) __builtin_amdgcn_s_waitcnt(0xc07f);  // this wave's codes are in registers: their place is free
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int now = k & 1;
      if (k == 3) {
        // younger than the loads of piece i + 1 are those of piece i + 2 and, where they began in this step or the last, those
        // of the weights
        if (!more_x) wait_loads<0>();
        else if (more_w) wait_loads<kRows + kW>();
        else wait_loads<kRows>();
        barrier();
        if (c == 3) read_w();
      }
#pragma unroll
      for (int j = 0; j < kParts; ++j) {
        const int m = j / WN, n = j % WN;
        acc[n][m] = Operand<TX>::mfma32(wv[now][n], xv[now][m], acc[n][m]);
        if (j == 0) {
          // all of the next step's rows at once: with the reads between the products, a product's wait for its own, which
          // counts from the oldest, took the newest with it
#pragma unroll
          for (int q = 0; q < kLive; ++q) read_x(k == 3 ? next : cur, k == 3 ? 0 : k + 1, now ^ 1, q);
          if constexpr (DIRECT)
            if (k == 0 && more_x) {
#pragma unroll
              for (int q = 0; q < kLive; ++q) load_x(old, i + 2, q);
            }
          if ((k == 1 || k == 2) && c == 0 && more_w) {
#pragma unroll
            for (int l = 0; l < kW; ++l)
              if (l * 2 / kW == k - 1) load_w(i / 4 + 1, l);
          }
        }
        // the next step's weights; a new part's as late as can be, they are being read
        if (j == (k == 3 && c == 3 ? kParts - 1 : (kParts - 1) / 2)) convert(k == 3 ? (c + 1) % 4 : c, (k + 1) % 4, now ^ 1);
        __builtin_amdgcn_sched_barrier(0);
      }
    }
  };
  auto run = [&](auto live) __attribute__((always_inline)) {
    constexpr int kLive = decltype(live)::value;
    if constexpr (DIRECT) {
#pragma unroll
      for (int m = 0; m < kLive; ++m) load_x(rows0, 0, m);
#pragma unroll
      for (int m = 0; m < kLive; ++m) load_x(rows1, min(1, pieces - 1), m);
    } else {
      fetch(0);
      put(rows0, 0);
      if (pieces > 1) {
        fetch(1);
        put(rows1, 1);
      }
      if (pieces > 2) fetch(2);
    }
    wait_loads<DIRECT ? kLive : 0>();
    __syncthreads();
    read_w();
#pragma unroll
    for (int m = 0; m < kLive; ++m) read_x(rows0, 0, 0, m);
    convert(0, 0, 0);
    using std::integral_constant;
    constexpr integral_constant<int, 0> c0{};
    constexpr integral_constant<int, 1> c1{};
    constexpr integral_constant<int, 2> c2{};
    constexpr integral_constant<int, 3> c3{};
    for (int i = 0; i < pieces; i += 12) {
      step(live, c0, rows2, rows0, rows1, i);
      if (i + 1 < pieces) step(live, c1, rows0, rows1, rows2, i + 1);
      if (i + 2 < pieces) step(live, c2, rows1, rows2, rows0, i + 2);
      if (i + 3 < pieces) step(live, c3, rows2, rows0, rows1, i + 3);
      if (i + 4 < pieces) step(live, c0, rows0, rows1, rows2, i + 4);
      if (i + 5 < pieces) step(live, c1, rows1, rows2, rows0, i + 5);
      if (i + 6 < pieces) step(live, c2, rows2, rows0, rows1, i + 6);
      if (i + 7 < pieces) step(live, c3, rows0, rows1, rows2, i + 7);
      if (i + 8 < pieces) step(live, c0, rows1, rows2, rows0, i + 8);
      if (i + 9 < pieces) step(live, c1, rows2, rows0, rows1, i + 9);
      if (i + 10 < pieces) step(live, c2, rows0, rows1, rows2, i + 10);
      if (i + 11 < pieces) step(live, c3, rows1, rows2, rows0, i + 11);
    }
  };
  const int tiles = (t.count + 31) / 32;
  static_assert(TM == 3, "a case for each number of tiles");
  if (tiles == 3) run(std::integral_constant<int, 3>{});
  else if (tiles == 2) run(std::integral_constant<int, 2>{});
  else run(std::integral_constant<int, 1>{});
  wait_loads<0>();
  __syncthreads();
  // Each wave turns its results, 32 rows at a time, into rows of the output's type in LDS and stores
  // them 16 bytes a lane: whole lines of the output.
  by_output(a, [&](auto to_type) {
    using TO = decltype(to_type);
    constexpr int kSize = ElemInfo<TO>::kBytes;
    constexpr int kPitch = WN * 32 * kSize + 16;  // 16 bytes more: the 32 rows start in different banks
    constexpr int kPerStage = kX / (32 * kPitch);
    // where a wave has two tiles of columns, they fit where its weights were; else where the rows were
    static_assert(WN == 2 ? 32 * kPitch <= (int)sizeof(weights[0]) : kPerStage * 3 >= W, "the buffers hold the results");
    uint8_t* mine = WN == 2 ? weights[wave]
                            : (wave / kPerStage == 0 ? rows0 : wave / kPerStage == 1 ? rows1 : rows2) +
                                  wave % kPerStage * (32 * kPitch);
#pragma unroll
    for (int m = 0; m < TM; ++m) {
      const int first = m * 32;
      if (first >= t.count) break;
      const bool dead = !row_live[first + l32];
      // lane l of a 32 x 32 result has row l % 32 and columns 8 * q + 4 * (l / 32) + 0..3, q = 0..3
#pragma unroll
      for (int n = 0; n < WN; ++n)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const int c = n * 32 + q * 8 + half * 4;
          float f[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            f[j] = (dead ? 0.f : acc[n][m][4 * q + j]) + col_bias[w0 + c + j];
            if (a.gelu) f[j] = gelu<TO>(f[j]);
          }
          apart<TO>(f);
          *reinterpret_cast<typename Vec<TO, 4>::raw_t*>(mine + l32 * kPitch + c * kSize) = Vec<TO, 4>::pack(f);
        }
      constexpr int kLanes = WN * 32 * kSize / 16;  // lanes of a row
      wave_order();
#pragma unroll
      for (int p = 0; p < 32 * kLanes / kWave; ++p) {
        const int r = p * (kWave / kLanes) + lane / kLanes, c = lane % kLanes * (16 / kSize);
        const u32x4 v = *reinterpret_cast<const u32x4*>(mine + r * kPitch + c * kSize);
        const int64_t n = n0 + w0 + c;
        if (first + r >= t.count || n >= a.N) continue;
        TO* to = static_cast<TO*>(a.out) + (t.row + first + r) * a.out_stride + n;
        if (n + 16 / kSize <= a.N) {
          *reinterpret_cast<u32x4_any*>(to) = v;
        } else {
          const int left = (int)(a.N - n);
#pragma unroll
          for (int j = 0; j < 16 / kSize; ++j)
            if (j < left) {
              if constexpr (kSize == 4) reinterpret_cast<uint32_t*>(to)[j] = v[j];
              else reinterpret_cast<uint16_t*>(to)[j] = (uint16_t)(v[j / 2] >> (16 * (j % 2)));
            }
        }
      }
      wave_order();  // the next tile's results go where these lay
    }
  });
}

// ---- weights to 4 bits and back ---------------------------------------------------------------------
// A thread takes the 32 weights of a scale: the smallest power of two with which none of them passes 6.  This is done once, when
// a layer is made: 64 experts' [2048, 4096] (1.36 GB with their bf16) take 0.96 ms, a launch and two copies for each, and back
// to bf16 in one launch 0.39 ms.
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

template <typename TX, int KS> int launch_few(const char* who, Fp4Args a, hipStream_t s) {
  const int64_t groups = grid_of(who, &a, 16, 16 * (kFewWaves / KS), kFewWaves * kWave);
  if (groups < 0) return FMOE_ERANGE;
  hipLaunchKernelGGL((k_fp4_few<TX, KS>), dim3((unsigned)groups), dim3(kFewWaves * kWave), 0, s, a);
  return fmoe_host::check_launch(who);
}

template <typename TX, int TM, int WN, bool AGAIN> int launch_tile(const char* who, Fp4Args a, hipStream_t s) {
  const int64_t groups = grid_of(who, &a, TM * 32, WN * 128, 4 * kWave);
  if (groups < 0) return FMOE_ERANGE;
  const bool direct = a.K % 64 == 0 && a.x_stride % 8 == 0 && reinterpret_cast<uintptr_t>(a.x) % 16 == 0;
  const dim3 grid((unsigned)groups), block(4 * kWave);
  if (direct) hipLaunchKernelGGL((k_fp4_tile<TX, TM, WN, true, AGAIN>), grid, block, 0, s, a);
  else hipLaunchKernelGGL((k_fp4_tile<TX, TM, WN, false, AGAIN>), grid, block, 0, s, a);
  return fmoe_host::check_launch(who);
}

// The variant for these sizes, as 1000 * rows + columns of its tile.  `per` is the rows of an expert were the routing even,
// tiles(bm) the tiles of bm rows that the experts then have, on the average over random routing.  Times in us of
// E experts' [N, K] at `per` rows each, by variant (16 x 128 / KS with K split over KS of the waves, 96 x 128, 96 x 256):
//                         16x128  16x64  16x32  16x16  96x128  96x256
//   1 [2048, 7168]    1    18.5    11.5     8.4    7.0    34.1    47.8
//                    16    27.9    23.6    17.8   14.9    36.0    51.4
//                    64    27.8    23.8    19.2   29.1    41.2    60.6
//   1 [7168, 2048]    1     8.3     7.5     6.6    9.4    14.8    19.2
//   8 [2048, 7168]    1    21.7    13.7    17.0   21.2    37.6    53.8
//                     8    28.6    20.5    32.5   48.9    39.2    56.4
//                    16    30.9    33.5    50.8   79.7    39.5    56.7
//                    32    46.8    52.8    90.8    142    43.1    62.7
//  64 [256, 2048]     1     8.5     7.2    10.5   14.6    15.2    19.2
//                    16    11.3    12.9    21.7   36.4    15.3    20.5
//                    64    25.3    30.1    66.5    110    19.2    28.3
//  16 [4096, 4096]    8    31.6    38.9    81.4    129    35.2    40.5
//                    16    55.1    62.2     133    220    36.1    40.7
//                   128     223     309     733   1208    97.2    82.4
//  32 [7168, 2048]    8    55.4    72.2     179    319    70.8    59.0
//                    16    83.6     118     302    524    71.3    61.3
// 256 [2048, 2048]    4     122     146     340    610     153     128
//                     8     126     163     420    731     153     123
//                    64     469     746    1964   3402     203     182
// A wave alone takes 0.55 us for 256 of K, so where there are few workgroups K is split until there are one or two on each
// CU; each workgroup brings all of its expert's rows, which a split multiplies.  Tiles of 96 rows take over where
// an expert's rows pass one tile of 16 (8 on the average), unless there are few workgroups even so; 256 columns from where
// they make more than one workgroup on a CU.
// The host knows how many rows there are, not whose.  Where one expert has most of them, its tiles of 16 read its weights
// again: 1024 rows of 256 experts' [2048, 2048] take 119 us evenly, 123 where one has 514 of them and 132 with 769; 512 of
// 64 experts' [2048, 4096] 64, 71 (260) and 78 (386); 256 of 32 experts' [7168, 2048] 58, 66 (132) and 70 (194).
enum Variant { k16x128 = 16128, k16x64 = 16064, k16x32 = 16032, k16x16 = 16016, k96x128 = 96128, k96x256 = 96256 };
Variant pick(int64_t rows, int64_t E, int64_t N) {
  const double per = (double)rows / (double)E;
  auto tiles = [&](double bm) {
    const double spread = E > 1 ? 2 * std::sqrt(per) : 0, least = std::ceil(std::max(per - spread, 0.0) / bm);
    const double more = E > 1 ? std::clamp((per + spread - least * bm) / (2 * spread), 0.0, 1.0) : 0.0;
    return std::min((double)E * (least + more), (double)rows);
  };
  const double few = tiles(16) * (double)((N + 127) / 128), wide = tiles(96) * (double)((N + 255) / 256);
  if (per <= 8 || few <= 280) {
    return few * 8 <= 256 ? k16x16 : few * 4 <= 256 ? k16x32 : few * 2 <= (per < 3 ? 640 : 300) ? k16x64 : k16x128;
  }
  return wide >= 288 && N > 128 ? k96x256 : k96x128;
}

template <typename TX> int launch_linear(const char* who, const Fp4Args& a, hipStream_t s) {
  switch (pick(a.rows, a.E, a.N)) {
    case k16x128: return launch_few<TX, 1>(who, a, s);
    case k16x64: return launch_few<TX, 2>(who, a, s);
    case k16x32: return launch_few<TX, 4>(who, a, s);
    case k16x16: return launch_few<TX, 8>(who, a, s);
    case k96x128: return launch_tile<TX, 3, 1, false>(who, a, s);
    default:
      // more than a tile's rows for many of the experts
      return a.rows > 80 * a.E ? launch_tile<TX, 3, 2, true>(who, a, s) : launch_tile<TX, 3, 2, false>(who, a, s);
  }
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

extern "C" int64_t fmoe_fp4_linear_tile(int64_t rows, int64_t num_experts, int64_t N, int64_t K) {
  if (rows < 1 || num_experts < 1 || N < 1 || K < 1) return -1;
  return pick(rows, num_experts, N);
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
                  num_experts, N, K, fmoe_host::round_up(K, kFp4Pitch), rows, d_out, out_row_stride, out_dtype, 0};
  hipStream_t s = static_cast<hipStream_t>(stream);
  return x_dtype == FMOE_BF16 ? launch_linear<bf16_t>(who, a, s) : launch_linear<f16_t>(who, a, s);
}
