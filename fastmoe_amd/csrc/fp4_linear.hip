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

// f(a value of the output's type)
template <typename F> __device__ __forceinline__ void by_output(const Fp4Args& a, F&& f) {
  if (a.out_dtype == FMOE_F32) f(float{});
  else if (a.out_dtype == FMOE_BF16) f(bf16_t{});
  else f(f16_t{});
}

// Few rows: 16 rows by 16 columns in a workgroup, whose eight waves take pieces of 128 of K in turn, straight from memory to
// the matrix units' registers, and add their parts in LDS in one order.
constexpr int kFp4Waves = 8;
template <typename TX> __global__ __launch_bounds__(kFp4Waves * kWave) void k_fp4_few(Fp4Args a) {
  __shared__ f32x4 part[kFp4Waves][kWave];
  Tile t;
  int group;
  if (!place<16>(a, &t, &group)) return;
  const int64_t n0 = (int64_t)group * 16;
  if (t.expert == a.E) {
    by_output(a, [&](auto to) { zero_rows<decltype(to)>(a, t, n0, 16); });
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
  by_output(a, [&](auto to) { store4<decltype(to)>(a, t, t.row + l16, n0 + quad * 4, acc); });
}

// BM rows by W * WN * 32 columns of one expert in a workgroup of W waves.  Each wave has every row and its own 32 WN
// columns, so each weight is converted once and a converted one serves all rows.  Pieces of 64 of K go through a
// ring of buffers in LDS, which the loads write directly where rows start at multiples of 16 bytes and K has whole pieces
// (DIRECT); else the rows' part goes through registers, zeros beyond K.
//
// In LDS a row's piece is 128 bytes, its 16-byte chunk c at position c ^ swizzle(row); an output's is 32 bytes, its
// halves exchanged in every other eight outputs: what a read's lanes touch together then lies in different banks.  Lane l of
// a matrix unit's operand has row (output) l % 32, and of a piece's K the half l / 32: four steps of 8.
// Scales lie in LDS for kWindow of K at a time; each wave brings its own outputs'.
constexpr int kWindow = 512;
template <typename TX, int BM, int W, int WN, int STAGES, bool DIRECT>
__global__ __launch_bounds__(W * kWave, 2) void k_fp4_tile(Fp4Args a) {
  constexpr int BN = W * WN * 32, TM = BM / 32;
  constexpr int kX = BM * 128, kStage = kX + BN * 32;
  constexpr int PX = BM / 8 / W, kLoads = (DIRECT ? PX : 0) + WN;  // loads of a wave a piece
  static_assert(PX * 8 * W == BM, "whole loads");
  static_assert(STAGES == 3 || STAGES == 4, "buffers");
  // separate objects: the compiler then sees that reads of one stage need not wait for the loads in
  // flight to the others
  __shared__ __attribute__((aligned(1024))) uint8_t stage0[kStage];
  __shared__ __attribute__((aligned(1024))) uint8_t stage1[kStage];
  __shared__ __attribute__((aligned(1024))) uint8_t stage2[kStage];
  __shared__ __attribute__((aligned(1024))) uint8_t stage3[STAGES > 3 ? kStage : 1];
  __shared__ uint32_t scales[BN][kWindow / kFp4Block / 4];
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
  const int w0 = wave * WN * 32;  // this wave's outputs
  const TX* xp[PX];
  int xc[PX];  // the column that the lane reads of a piece
#pragma unroll
  for (int i = 0; i < PX; ++i) {
    const int r = (wave * PX + i) * 8 + lane / 8;
    xp[i] = static_cast<const TX*>(a.x) + max(source_row(a, t.row + min(r, t.count - 1)), (int64_t)0) * a.x_stride;
    xc[i] = (lane % 8 ^ swizzle<128>(r)) * 8;
    if constexpr (DIRECT) xp[i] += xc[i];
  }
  const uint8_t* wp[WN];
#pragma unroll
  for (int i = 0; i < WN; ++i) {
    const int c = lane / 2;
    const int64_t col = t.expert * a.N + min(n0 + w0 + i * 32 + c, a.N - 1);
    wp[i] = a.w + col * (a.Kp / 2) + ((lane & 1) ^ (c >> 3 & 1)) * 16;
  }
  const int pieces = (int)((a.K + 63) / 64);
  // loads beyond the last piece read it once more, into a buffer that nobody reads: the number of
  // loads in flight is then the same in every step
  auto at = [&](int piece) { return (int64_t)min(piece, pieces - 1); };
  auto load_one = [&](uint8_t* s, int64_t piece, int i) {
    if (DIRECT && i < PX)
      load_piece<kCPolCached>(reinterpret_cast<const uint8_t*>(xp[i < PX ? i : 0] + piece * 64), s + (wave * PX + i) * 1024);
    else {
      const int j = i - (DIRECT ? PX : 0);
      load_piece<kCPolCached>(wp[j] + piece * 32, s + kX + (wave * WN + j) * 1024);
    }
  };
  u32x4 xr[DIRECT ? 1 : PX];  // the rows' part of a piece on its way
  auto fetch = [&](int64_t piece) {
    if constexpr (!DIRECT)
#pragma unroll
      for (int i = 0; i < PX; ++i) xr[i] = Eight<TX>::template load<false>(xp[i], piece * 64 + xc[i], a.K);
  };
  auto put = [&](uint8_t* s) {
    if constexpr (!DIRECT)
#pragma unroll
      for (int i = 0; i < PX; ++i) *reinterpret_cast<u32x4*>(s + (wave * PX + i) * 1024 + lane * 16) = xr[i];
  };
  // this wave's scales from column `k` on, an output's 16 bytes in four lanes
  const uint8_t* sp = a.s + t.expert * a.N * (a.Kp / kFp4Block);
  auto window = [&](int64_t k) {
    const int64_t Ks = a.Kp / kFp4Block, from = k / kFp4Block + lane % 4 * 4;
#pragma unroll
    for (int i = 0; i < WN * 2; ++i) {
      const int c = w0 + i * 16 + lane / 4;
      scales[c][lane % 4] = *reinterpret_cast<const uint32_t*>(sp + min(n0 + c, a.N - 1) * Ks + min(from, Ks - 4));
    }
    wave_order();
  };
  f32x16 acc[WN][TM];
#pragma unroll
  for (int n = 0; n < WN; ++n)
#pragma unroll
    for (int m = 0; m < TM; ++m)
#pragma unroll
      for (int i = 0; i < 16; ++i) acc[n][m][i] = 0.f;
  u32x4 xv[2][TM], wv[2][WN];  // operands of this and the next step
  u32x4 codes[WN], next_codes[WN];
  float scale[WN], next_scale[WN];
  auto read_x = [&](const uint8_t* s, int k, int to, int m) {
    xv[to][m] = *reinterpret_cast<const u32x4*>(s + (m * 32 + l32) * 128 + ((half * 4 + k) ^ swizzle<128>(l32)) * 16);
  };
  auto read_codes = [&](const uint8_t* s, u32x4* to) {
#pragma unroll
    for (int n = 0; n < WN; ++n)
      to[n] = *reinterpret_cast<const u32x4*>(s + kX + (w0 + n * 32 + l32) * 32 + (half ^ (l32 >> 3 & 1)) * 16);
  };
  auto read_scales = [&](int piece, float* to) {
#pragma unroll
    for (int n = 0; n < WN; ++n) {
      const uint8_t* four = reinterpret_cast<const uint8_t*>(scales[w0 + n * 32 + l32]);
      to[n] = __uint_as_float((uint32_t)four[piece % (kWindow / 64) * 2 + half] << 23);
    }
  };
  // Step i multiplies piece i in buffer `cur`, by `live` tiles of 32 rows.  Before its last part each wave has read all of
  // the piece and waits until its loads of piece i + 1 have arrived; behind the barrier that holds for every
  // wave, so `next` is read, and `cur` is free.  Piece i + STAGES - 1 is loaded into `old`.
  auto step = [&](auto live, uint8_t* old, uint8_t* cur, const uint8_t* next, int i)
                  __attribute__((always_inline)) {
    constexpr int kLive = decltype(live)::value;
    const int64_t rest = at(i + STAGES - 1);
    if ((i + 1) % (kWindow / 64) == 0 && i + 1 < pieces) window((int64_t)(i + 1) * 64);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int now = k & 1;
      if (k == 0) {
        put(old);  // what was fetched in the last step
        fetch(at(i + STAGES));
      }
      if (k == 1) read_scales(i + 1, next_scale);
      if (k == 3) {
        wait_loads<(STAGES - 2) * kLoads>();
        barrier();
        read_codes(next, next_codes);
      }
      constexpr int kOps = kLive;
#pragma unroll
      for (int j = 0; j < kLive * WN; ++j) {
        const int m = j / WN, n = j % WN;
        acc[n][m] = Operand<TX>::mfma32(wv[now][n], xv[now][m], acc[n][m]);
#pragma unroll
        for (int o = j * kOps / (kLive * WN); o < (j + 1) * kOps / (kLive * WN); ++o)
          read_x(k == 3 ? next : cur, k == 3 ? 0 : k + 1, now ^ 1, o);
        if (k < 3) {
#pragma unroll
          for (int l = kLoads * (k * kLive * WN + j) / (3 * kLive * WN); l < kLoads * (k * kLive * WN + j + 1) / (3 * kLive * WN); ++l)
            load_one(old, rest, l);
        }
        // the next step's weights: of the next piece as late as can be, its codes were asked for in this step
        constexpr int kLast = kLive * WN - 1;
        if (j == (k == 3 ? kLast : kLast / 2)) {
#pragma unroll
          for (int q = 0; q < WN; ++q)
            wv[now ^ 1][q] = k == 3 ? Operand<TX>::weights(next_codes[q][0], next_scale[q])
                                    : Operand<TX>::weights(codes[q][(k + 1) % 4], scale[q]);
        }
        __builtin_amdgcn_sched_barrier(0);
      }
    }
#pragma unroll
    for (int n = 0; n < WN; ++n) {
      codes[n] = next_codes[n];
      scale[n] = next_scale[n];
    }
  };
  auto run = [&](auto live) __attribute__((always_inline)) {
    int i = 0;
    if constexpr (STAGES == 3) {
      for (; i + 3 <= pieces; i += 3) {
        step(live, stage2, stage0, stage1, i);
        step(live, stage0, stage1, stage2, i + 1);
        step(live, stage1, stage2, stage0, i + 2);
      }
      if (i < pieces) step(live, stage2, stage0, stage1, i);
      if (i + 1 < pieces) step(live, stage0, stage1, stage2, i + 1);
    } else {
      for (; i + 4 <= pieces; i += 4) {
        step(live, stage3, stage0, stage1, i);
        step(live, stage0, stage1, stage2, i + 1);
        step(live, stage1, stage2, stage3, i + 2);
        step(live, stage2, stage3, stage0, i + 3);
      }
      if (i < pieces) step(live, stage3, stage0, stage1, i);
      if (i + 1 < pieces) step(live, stage0, stage1, stage2, i + 1);
      if (i + 2 < pieces) step(live, stage1, stage2, stage3, i + 2);
    }
  };
  auto ring = [&](int i) { return i == 0 ? stage0 : i == 1 ? stage1 : i == 2 ? stage2 : stage3; };
  for (int c = threadIdx.x; c < BN; c += W * kWave)
    col_bias[c] = a.bias ? load_weight(a.bias, a.bias_dtype, t.expert * a.N + min(n0 + c, a.N - 1)) : 0.f;
  for (int r = threadIdx.x; r < BM; r += W * kWave) row_live[r] = source_row(a, t.row + min(r, t.count - 1)) >= 0;
  window(0);
#pragma unroll
  for (int i = 0; i < STAGES - 1; ++i) {
    fetch(at(i));
    put(ring(i));
#pragma unroll
    for (int l = 0; l < kLoads; ++l) load_one(ring(i), at(i), l);
  }
  fetch(at(STAGES - 1));
  wait_loads<(STAGES - 2) * kLoads>();
  __syncthreads();
  read_codes(stage0, codes);
  read_scales(0, scale);
#pragma unroll
  for (int m = 0; m < TM; ++m) read_x(stage0, 0, 0, m);
#pragma unroll
  for (int n = 0; n < WN; ++n) wv[0][n] = Operand<TX>::weights(codes[n][0], scale[n]);
  const int tiles = (t.count + 31) / 32;
  if constexpr (TM == 1) run(std::integral_constant<int, 1>{});
  else if constexpr (TM == 2) {
    if (tiles == 1) run(std::integral_constant<int, 1>{});
    else run(std::integral_constant<int, 2>{});
  } else {
    if (tiles == 1) run(std::integral_constant<int, 1>{});
    else if (tiles == 2) run(std::integral_constant<int, 2>{});
    else if (tiles == 3) run(std::integral_constant<int, 3>{});
    else run(std::integral_constant<int, 4>{});
  }
  wait_loads<0>();
  __syncthreads();
  // Each wave turns its results, 32 rows at a time, into rows of the output's type in LDS and stores
  // them 16 bytes a lane: whole lines of the output.
  by_output(a, [&](auto to_type) {
    using TO = decltype(to_type);
    constexpr int kSize = ElemInfo<TO>::kBytes;
    constexpr auto fits = [](int tiles) { return kStage / (32 * (tiles * 32 * kSize + 16)) * STAGES >= W; };
    constexpr int CT = fits(WN) ? WN : 1;  // column tiles at a time
    constexpr int kPitch = CT * 32 * kSize + 16;  // 16 bytes more: the 32 rows start in different banks
    constexpr int kPerStage = kStage / (32 * kPitch);
    static_assert(kPerStage * STAGES >= W, "the stages hold the results");
    uint8_t* mine = ring(wave / kPerStage) + wave % kPerStage * (32 * kPitch);
#pragma unroll
    for (int m = 0; m < TM; ++m) {
      const int first = m * 32;
      if (first >= t.count) break;
      const bool dead = !row_live[first + l32];
      // lane l of a 32 x 32 result has row l % 32 and columns 8 * q + 4 * (l / 32) + 0..3, q = 0..3
#pragma unroll
      for (int base = 0; base < WN; base += CT) {
#pragma unroll
        for (int n = 0; n < CT; ++n)
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const int c = n * 32 + q * 8 + half * 4;
            float f[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              f[j] = (dead ? 0.f : acc[base + n][m][4 * q + j]) + col_bias[w0 + base * 32 + c + j];
              if (a.gelu) f[j] = gelu<TO>(f[j]);
            }
            apart<TO>(f);
            *reinterpret_cast<typename Vec<TO, 4>::raw_t*>(mine + l32 * kPitch + c * kSize) = Vec<TO, 4>::pack(f);
          }
        constexpr int kLanes = CT * 32 * kSize / 16;  // lanes of a row
        wave_order();
#pragma unroll
        for (int p = 0; p < 32 * kLanes / kWave; ++p) {
          const int r = p * (kWave / kLanes) + lane / kLanes, c = lane % kLanes * (16 / kSize);
          const u32x4 v = *reinterpret_cast<const u32x4*>(mine + r * kPitch + c * kSize);
          const int64_t n = n0 + w0 + base * 32 + c;
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
        wave_order();  // the next tiles' results go where these lay
      }
    }
  });
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

template <typename TX> int launch_few(const char* who, Fp4Args a, hipStream_t s) {
  const int64_t groups = grid_of(who, &a, 16, 16, kFp4Waves * kWave);
  if (groups < 0) return FMOE_ERANGE;
  hipLaunchKernelGGL((k_fp4_few<TX>), dim3((unsigned)groups), dim3(kFp4Waves * kWave), 0, s, a);
  return fmoe_host::check_launch(who);
}

template <typename TX, int BM, int W, int WN, int STAGES>
int launch_tile(const char* who, Fp4Args a, hipStream_t s) {
  const int64_t groups = grid_of(who, &a, BM, W * WN * 32, W * kWave);
  if (groups < 0) return FMOE_ERANGE;
  const bool direct = a.K % 64 == 0 && a.x_stride % 8 == 0 && reinterpret_cast<uintptr_t>(a.x) % 16 == 0;
  const dim3 grid((unsigned)groups), block(W * kWave);
  if (direct) hipLaunchKernelGGL((k_fp4_tile<TX, BM, W, WN, STAGES, true>), grid, block, 0, s, a);
  else hipLaunchKernelGGL((k_fp4_tile<TX, BM, W, WN, STAGES, false>), grid, block, 0, s, a);
  return fmoe_host::check_launch(who);
}

// The variant for these sizes, as 1000 * rows + columns of its tile.
enum Variant { kFew = 16016, k32x128 = 32128, k64x128 = 64128, k128x256 = 128256 };
#ifndef FMOE_FP4_TILE
#define FMOE_FP4_TILE 0
#endif
Variant pick(int64_t rows, int64_t E, int64_t N, int64_t K) {
  if (FMOE_FP4_TILE) return (Variant)FMOE_FP4_TILE;
  const int64_t per = rows / E;
  if (per <= 8) return kFew;
  if (per <= 32) return k32x128;
  if (per <= 64) return k64x128;
  return k128x256;
}

template <typename TX> int launch_linear(const char* who, const Fp4Args& a, hipStream_t s) {
  switch (pick(a.rows, a.E, a.N, a.K)) {
    case k32x128: return launch_tile<TX, 32, 4, 1, 4>(who, a, s);
    case k64x128: return launch_tile<TX, 64, 4, 1, 4>(who, a, s);
    case k128x256: return launch_tile<TX, 128, 4, 2, 3>(who, a, s);
    default: return launch_few<TX>(who, a, s);
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
  return pick(rows, num_experts, N, K);
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
