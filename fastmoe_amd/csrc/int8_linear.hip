// Every expert's product on its own rows, in 8-bit integers:
//
//   out[r, n] = (sum_k x[i(r), k] * w[e(r), n, k]) * sx[i(r)] * sw[e(r), n] + b[e(r), n]
//
// for packed rows r in [off[e], off[e + 1]) of expert e; i(r) = index[r] where the rows are read
// through an index (the dispatch's reverse map: the rows of a token are never copied for its
// experts), else r.  The sums are int32 and exact (K <= 131071 keeps them in range: 128 * 128 * K <
// 2^31), so neither the order nor a split of K changes a bit; each is then converted to fp32 once
// (2^-24), scaled and rounded to the output's type.  A row's scale below one is multiplied first and
// a larger one last: then no step overflows or vanishes unless the result does (rows near the largest
// numbers have scales up to 2^121, which times the sum would be infinite whatever the weights').  The last
// factor comes with the bias' addition, in one instruction.
//
// Rows and weights lie with K innermost, padded with zeros to whole pieces of 128 bytes, so no
// product needs a tail in K.  Rows of a tile beyond its expert's last repeat that last one, columns
// beyond N repeat the last one; neither is stored.
#include "expert_tiles.h"

#include <algorithm>
#include <cmath>

namespace fmoe {

struct LinearArgs {
  const uint8_t* x;       // 8-bit rows
  int64_t x_stride;       // bytes
  int64_t x_rows;
  const float* sx;        // [x_rows]
  const void* index;      // [rows], or null: row r reads row r
  int index_dtype;
  const uint8_t* w;       // [E, N, Kp]
  const float* sw;        // [E, N]
  const void* bias;       // [E, N], or null
  int bias_dtype;
  const int64_t* off;     // [E + 1], or null: one expert has every row
  int64_t E, N, Kp, rows;
  void* out;
  int64_t out_stride;     // elements
  int groups_n;           // workgroups side by side that cover N
};

// A row's scale as the factors before and after the output's scale.
struct RowScale {
  float before, after;
  __device__ __forceinline__ explicit RowScale(float s)
      : before(__builtin_fabsf(s) < 1.f ? s : 1.f), after(__builtin_fabsf(s) < 1.f ? 1.f : s) {}  // NaN: after
  __device__ __forceinline__ float scaled(int32_t sum, float sw, float bias) const {
    return __builtin_fmaf((float)sum * before * sw, after, bias);
  }
};

// Four neighbouring columns of one output row.
template <typename TO>
__device__ __forceinline__ void store4(const LinearArgs& a, const Tile& t, int64_t r, int64_t n,
                                       i32x4 acc, RowScale sx) {
  if (n >= a.N) return;
  TO* p = static_cast<TO*>(a.out) + r * a.out_stride + n;
  float f[4];
  const float* sw = a.sw + t.expert * a.N + n;
  const int left = (int)min((int64_t)4, a.N - n);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    f[i] = 0.f;
    if (i < left) {
      const float bias = a.bias ? load_weight(a.bias, a.bias_dtype, t.expert * a.N + n + i) : 0.f;
      f[i] = sx.scaled(acc[i], sw[i], bias);
    }
  }
  apart<TO>(f);
  if (left == 4) {
    if constexpr (ElemInfo<TO>::kBytes == 4)
      *reinterpret_cast<u32x4_any*>(p) = Vec<TO, 4>::pack(f);
    else
      *reinterpret_cast<u32x2_any*>(p) = Vec<TO, 4>::pack(f);
  } else {
    for (int i = 0; i < left; ++i) st1(p + i, f[i]);
  }
}

// Few rows and few columns: 16 x 16 results in a workgroup, whose eight waves take 128-byte pieces of K
// in turn, straight from memory to the matrix units' registers, and add their int32 parts in LDS.
// Where even the smallest tile below leaves most CUs without work, splitting K over the waves is what is
// left: 9.2 against 19 us for one row and [2048, 7168] weights, 32 workgroups of 32 x 64 (but 27.9
// against 25.1 us with eight experts' weights, 256 workgroups).
constexpr int kFewWaves = 8;
template <typename TO> __global__ __launch_bounds__(kFewWaves * kWave) void k_int8_few(LinearArgs a) {
  __shared__ i32x4 part[kFewWaves][kWave];
  Tile t;
  int group;
  if (!place<16>(a, &t, &group)) return;
  const int64_t n0 = (int64_t)group * 16;
  if (t.expert == a.E) {
    zero_rows<TO>(a, t, n0, 16);
    return;
  }
  const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
  const int l16 = lane & 15, quad = lane >> 4;
  const int64_t row = source_row(a, t.row + min(l16, t.count - 1));
  const uint8_t* xp = a.x + max(row, (int64_t)0) * a.x_stride + quad * 16;
  const uint8_t* wp = a.w + (t.expert * a.N + min(n0 + l16, a.N - 1)) * a.Kp + quad * 16;
  i32x4 acc = {0, 0, 0, 0};
  constexpr int kStep = kFewWaves * 128, kAhead = 4;  // pieces asked for before the first is used
  auto pieces = [&](auto count, int64_t k) {
    constexpr int n = 2 * decltype(count)::value;
    i32x4 w[n], x[n];
#pragma unroll
    for (int i = 0; i < n; ++i) {
      const int64_t at = k + i / 2 * kStep + i % 2 * 64;
      w[i] = __builtin_nontemporal_load(reinterpret_cast<const i32x4*>(wp + at));
      x[i] = *reinterpret_cast<const i32x4*>(xp + at);
    }
#pragma unroll
    for (int i = 0; i < n; ++i) acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(w[i], x[i], acc, 0, 0, 0);
  };
  int64_t k = wave * 128;
  for (; k + (kAhead - 1) * kStep < a.Kp; k += kAhead * kStep)
    pieces(std::integral_constant<int, kAhead>{}, k);
  for (; k < a.Kp; k += kStep) pieces(std::integral_constant<int, 1>{}, k);
  part[wave][lane] = acc;
  __syncthreads();
  if (wave != 0 || l16 >= t.count) return;
#pragma unroll
  for (int v = 1; v < kFewWaves; ++v) acc += part[v][lane];
  // lane l of a 16 x 16 result has row l % 16 and columns 4 * (l / 16) + 0..3
  store4<TO>(a, t, t.row + l16, n0 + quad * 4, acc, RowScale(row >= 0 ? a.sx[row] : 0.f));
}

// BM x BN results of one expert in a workgroup of WR x WC waves, each wave (BM / WR) x (BN / WC) of them in
// its registers as 32 x 32 tiles.  Pieces of KB bytes of K of both operands go through a ring of
// STAGES buffers in LDS, which the loads write directly (no registers, no LDS store instructions).
//
// A row's 16-byte chunks lie in LDS at position chunk ^ swizzle(row): memory is read in whole pieces of
// a row, and the rows that the lanes of a fragment's read touch together lie in different banks
// (64 banks of 4 bytes: 256 / KB rows fill them once).
typedef int32_t i32x16 __attribute__((ext_vector_type(16)));
template <typename TO, int BM, int BN, int WR, int WC, int KB, int STAGES, bool EARLY, int CPOL, bool PAST>
__global__ __launch_bounds__(WR * WC * kWave) void k_int8_tile(LinearArgs a) {
  constexpr int kWaves = WR * WC;
  constexpr int TM = BM / WR / 32, TN = BN / WC / 32;  // 32 x 32 tiles of a wave
  constexpr int kRows = 1024 / KB;                     // rows of one load of a wave
  constexpr int PX = BM / kRows / kWaves, PW = BN / kRows / kWaves, kLoads = PX + PW;
  constexpr int kStage = (BM + BN) * KB, kSteps = KB / 32;
  static_assert(STAGES == 3 || STAGES == 4, "buffers");
  static_assert(PX * kRows * kWaves == BM && PW * kRows * kWaves == BN, "whole loads");
  // separate objects: the compiler then sees that reads of one stage need not wait for the loads in
  // flight to the others
  __shared__ __attribute__((aligned(1024))) uint8_t stage0[kStage];
  __shared__ __attribute__((aligned(1024))) uint8_t stage1[kStage];
  __shared__ __attribute__((aligned(1024))) uint8_t stage2[kStage];
  __shared__ __attribute__((aligned(1024))) uint8_t stage3[STAGES > 3 ? kStage : 1];
  __shared__ float row_scale[BM], col_scale[BN], col_bias[BN];
  Tile t;
  int group;
  if (!place<BM>(a, &t, &group)) return;
  const int64_t n0 = (int64_t)group * BN;
  if (t.expert == a.E) {
    zero_rows<TO>(a, t, n0, BN);
    return;
  }
  const int lane = threadIdx.x & (kWave - 1), wave = uniform(threadIdx.x / kWave);
  const uint8_t *xp[PX], *wp[PW];
#pragma unroll
  for (int i = 0; i < PX; ++i) {
    const int r = (wave * PX + i) * kRows + lane / (KB / 16);
    xp[i] = a.x + max(source_row(a, t.row + min(r, t.count - 1)), (int64_t)0) * a.x_stride +
            (lane % (KB / 16) ^ swizzle<KB>(r)) * 16;
  }
#pragma unroll
  for (int i = 0; i < PW; ++i) {
    const int r = (wave * PW + i) * kRows + lane / (KB / 16);
    wp[i] = a.w + (t.expert * a.N + min(n0 + r, a.N - 1)) * a.Kp +
            (lane % (KB / 16) ^ swizzle<KB>(r)) * 16;
  }
  auto load_one = [&](uint8_t* s, int64_t at, int i) {
    if (i < PX) load_piece<kCPolCached>(xp[i < PX ? i : 0] + at, s + (wave * PX + i) * 1024);
    else load_piece<CPOL>(wp[i < PX ? 0 : i - PX] + at, s + BM * KB + (wave * PW + i - PX) * 1024);
  };
  auto load = [&](uint8_t* s, int64_t at) {
#pragma unroll
    for (int i = 0; i < kLoads; ++i) load_one(s, at, i);
  };
  i32x16 acc[TN][TM];
#pragma unroll
  for (int n = 0; n < TN; ++n)
#pragma unroll
    for (int m = 0; m < TM; ++m)
#pragma unroll
      for (int i = 0; i < 16; ++i) acc[n][m][i] = 0;
  const int l32 = lane & 31, half = lane >> 5;
  // the waves of a SIMD (every fourth) have different rows: where a tile's last rows are missing, the
  // matrix units are shared by the waves that have rows
  const int m0 = (wave / WC) * (BM / WR), w0 = (wave % WC) * (BN / WC);
  const bool busy = m0 < t.count;
  // fragments of 32 bytes of K: lane l has row l % 32 and bytes 16 * (l / 32) + 0..15
  i32x4 xv[2][TM], wv[2][TN];
  auto read_one = [&](const uint8_t* s, int k, int to, int i) {
    const int at = ((2 * k + half) ^ swizzle<KB>(l32)) * 16 + l32 * KB;
    if (i < TM)
      xv[to][i < TM ? i : 0] = *reinterpret_cast<const i32x4*>(s + (m0 + i * 32) * KB + at);
    else
      wv[to][i < TM ? 0 : i - TM] =
          *reinterpret_cast<const i32x4*>(s + (BM + w0 + (i - TM) * 32) * KB + at);
  };
  const int pieces = (int)(a.Kp / KB);
  // loads beyond the last piece read it once more, into a buffer that nobody reads: the number of
  // loads in flight is then the same in every step
  auto at = [&](int piece) { return (int64_t)min(piece, pieces - 1) * KB; };
  // Step i multiplies piece i in buffer `cur`.  Before its last fragments are multiplied, each wave has
  // read all of the piece and waits until its loads of piece i + 1 have arrived; behind the barrier that
  // holds for every wave, so `next` is read, and `cur` is free for piece i + STAGES.  EARLY: that piece's
  // loads begin there and end before the next barrier (so step i first goes on with piece
  // i + STAGES - 1 into `old`).  Else they begin with the next step, spread over all of it.  Tiles that
  // wait for memory gain by more in flight (128 rows over 256 experts of [2048, 7168], 32 x 128: 230 us,
  // else 249; 8 rows, 32 x 64: 22.7 and 25.2; 2048 rows over 32 experts of [7168, 2048], 128 x 256: 107.2
  // and 109.7), the others nothing (128 x 128: 37.7 and 37.4 at 384 rows over 8 experts of
  // [4096, 4096]; 256 x 256: 471 to 473 us either way at 49152 rows over 64 experts of [2048, 4096]).
  // Reads and loads stand between the products, one or two at a time: issued together they would hold
  // the wave back while the matrix units run dry.
  constexpr auto part = [](int k) { return k * kLoads / kSteps; };  // loads before part k of a piece's
  auto step = [&](auto works, uint8_t* old, uint8_t* cur, const uint8_t* next, int i) {
    const int64_t rest = at(i + STAGES - 1), from = at(i + STAGES);
#pragma unroll
    for (int k = 0; k < kSteps; ++k) {
      const bool last = k + 1 == kSteps, ahead = EARLY && last;
      if (last) {
        wait_loads<EARLY ? (STAGES - 2) * kLoads : (STAGES - 3) * kLoads + part(kSteps - 1)>();
        barrier();
      }
      const int p = !EARLY ? k : last ? 0 : k + 1;
      const int first = part(p), more = part(p + 1) - first;
      auto load_next = [&](int o) { load_one(ahead ? cur : old, ahead ? from : rest, first + o); };
      if constexpr (decltype(works)::value) {
        constexpr int kOps = TM + TN;
        const int ops = kOps + more;
#pragma unroll
        for (int j = 0; j < TM * TN; ++j) {
          acc[j / TM][j % TM] = __builtin_amdgcn_mfma_i32_32x32x32_i8(
              wv[k & 1][j / TM], xv[k & 1][j % TM], acc[j / TM][j % TM], 0, 0, 0);
#pragma unroll
          for (int o = j * ops / (TM * TN); o < (j + 1) * ops / (TM * TN); ++o) {
            if (o < kOps) read_one(last ? next : cur, last ? 0 : k + 1, (k + 1) & 1, o);
            else load_next(o - kOps);
          }
          __builtin_amdgcn_sched_barrier(0);
        }
      } else {  // no rows for this wave: it only loads its share
#pragma unroll
        for (int o = 0; o < more; ++o) load_next(o);
      }
    }
  };
  auto run = [&](auto works) {
    int i = 0;
    if constexpr (STAGES == 3) {
      for (; i + 3 <= pieces; i += 3) {
        step(works, stage2, stage0, stage1, i);
        step(works, stage0, stage1, stage2, i + 1);
        step(works, stage1, stage2, stage0, i + 2);
      }
      if (i < pieces) step(works, stage2, stage0, stage1, i);
      if (i + 1 < pieces) step(works, stage0, stage1, stage2, i + 1);
    } else {
      for (; i + 4 <= pieces; i += 4) {
        step(works, stage3, stage0, stage1, i);
        step(works, stage0, stage1, stage2, i + 1);
        step(works, stage1, stage2, stage3, i + 2);
        step(works, stage2, stage3, stage0, i + 3);
      }
      if (i < pieces) step(works, stage3, stage0, stage1, i);
      if (i + 1 < pieces) step(works, stage0, stage1, stage2, i + 1);
      if (i + 2 < pieces) step(works, stage1, stage2, stage3, i + 2);
    }
  };
  load(stage0, at(0));
  __builtin_amdgcn_sched_barrier(0);
  // the rows' scales, the columns' scales and biases: asked for here, so that they arrive between the
  // first pieces, and used at the end
  static_assert(BM <= kWaves * kWave && BN <= kWaves * kWave, "a row and a column for each thread");
  const int64_t my_row = source_row(a, t.row + min((int)threadIdx.x, t.count - 1));
  const int64_t my_col = t.expert * a.N + min(n0 + threadIdx.x, a.N - 1);
  const float my_row_scale = a.sx[max(my_row, (int64_t)0)];
  const float my_col_scale = a.sw[my_col];
  const float my_bias = a.bias ? load_weight(a.bias, a.bias_dtype, my_col) : 0.f;
  __builtin_amdgcn_sched_barrier(0);
  load(stage1, at(1));
  if constexpr (STAGES > 3) load(stage2, at(2));
  __builtin_amdgcn_sched_barrier(0);
  if (threadIdx.x < BM) row_scale[threadIdx.x] = my_row >= 0 ? my_row_scale : 0.f;
  if (threadIdx.x < BN) {
    col_scale[threadIdx.x] = my_col_scale;
    col_bias[threadIdx.x] = my_bias;
  }
  constexpr int kBegun = EARLY ? part(1) : 0;  // loads of piece STAGES - 1
#pragma unroll
  for (int i = 0; i < kBegun; ++i) load_one(STAGES > 3 ? stage3 : stage2, at(STAGES - 1), i);
  wait_loads<(STAGES - 2) * kLoads + kBegun>();
  barrier();
#pragma unroll
  for (int i = 0; i < TM + TN; ++i) read_one(stage0, 0, 0, i);
  if (busy) run(std::true_type{});
  else run(std::false_type{});
  wait_loads<0>();
  __syncthreads();
  // Each wave turns its results, 32 rows at a time, into rows of the output's type in LDS and stores
  // them 16 bytes a lane: whole lines of the output.
  constexpr int kSize = ElemInfo<TO>::kBytes;
  // column tiles at a time: as many as the stages hold for every wave
  constexpr auto fits = [](int tiles) {
    return kStage / (32 * (tiles * 32 * kSize + 16)) * STAGES >= kWaves;
  };
  constexpr int CT = fits(TN) ? TN : fits(TN / 2) ? TN / 2 : TN / 4;
  constexpr int kPitch = CT * 32 * kSize + 16;  // 16 bytes more: the 32 rows start in different banks
  constexpr int kPerStage = kStage / (32 * kPitch);
  static_assert(kPerStage * STAGES >= kWaves, "the stages hold the results");
  const int place_in = wave / kPerStage;
  uint8_t* mine = (place_in == 0 ? stage0 : place_in == 1 ? stage1 : place_in == 2 ? stage2 : stage3) +
                  wave % kPerStage * (32 * kPitch);
#pragma unroll
  for (int m = 0; m < TM; ++m) {
    const int first = m0 + m * 32;
    if (first >= t.count) break;
    const RowScale sx(row_scale[first + l32]);
    // lane l of a 32 x 32 result has row l % 32 and columns 8 * q + 4 * (l / 32) + 0..3, q = 0..3
#pragma unroll
    for (int base = 0; base < TN; base += CT) {
#pragma unroll
      for (int n = 0; n < CT; ++n)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const int c = n * 32 + q * 8 + half * 4;
          const int at_col = w0 + base * 32 + c;
          float f[4];
#pragma unroll
          for (int j = 0; j < 4; ++j)
            f[j] = sx.scaled(acc[base + n][m][4 * q + j], col_scale[at_col + j], col_bias[at_col + j]);
          apart<TO>(f);
          *reinterpret_cast<typename Vec<TO, 4>::raw_t*>(mine + l32 * kPitch + c * kSize) =
              Vec<TO, 4>::pack(f);
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
          if constexpr (PAST) __builtin_nontemporal_store(v, reinterpret_cast<u32x4_any*>(to));
          else *reinterpret_cast<u32x4_any*>(to) = v;
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
}

}  // namespace fmoe

using namespace fmoe;

namespace {

constexpr int64_t kMaxK = 131071;

template <typename TO> int launch_few(const char* who, LinearArgs a, hipStream_t s) {
  const int64_t groups = grid_of(who, &a, 16, 16, kFewWaves * kWave);
  if (groups < 0) return FMOE_ERANGE;
  hipLaunchKernelGGL(k_int8_few<TO>, dim3((unsigned)groups), dim3(kFewWaves * kWave), 0, s, a);
  return fmoe_host::check_launch(who);
}

template <typename TO, int BM, int BN, int WR, int WC, int KB, int STAGES, bool EARLY, int CPOL,
          bool PAST = (BN >= 256)>
int launch_tile(const char* who, LinearArgs a, hipStream_t s) {
  const int64_t groups = grid_of(who, &a, BM, BN, WR * WC * kWave);
  if (groups < 0) return FMOE_ERANGE;
  hipLaunchKernelGGL((k_int8_tile<TO, BM, BN, WR, WC, KB, STAGES, EARLY, CPOL, PAST>),
                     dim3((unsigned)groups), dim3(WR * WC * kWave), 0, s, a);
  return fmoe_host::check_launch(who);
}

// The variant for these sizes: the largest tile that the experts' rows fill and that leaves no CU
// without work.  `per` is the rows of an expert were the routing even, work(bm, bn) the workgroups then.
// Times in us of 32 experts' [2048, 7168] weights / 128 experts' [1024, 2048] / 8 experts' [4096, 4096]:
//   rows per expert     1              4              16             48              128            256
//   16 x 16 (few)  70 / 58 / 27  110 / 83 / 37  191 / 137 / 60  431 / 300 / 136
//   32 x 64        52 / 35 / 24   78 / 51 / 31   82 / 55 / 31   156 / 104 / 50  301 / 181 / 90  582 / 327 / 159
//   32 x 128       57 / 37 / 26   72 / 45 / 32   74 / 51 / 32   124 / 90 / 38   245 / 157 / 79  481 / 285 / 134
//   128 x 128      80 / 45 / 31   90 / 56 / 36   94 / 59 / 36   102 / 65 / 37   151 / 95 / 56   234 / 144 / 76
//   128 x 256      58 / 42 / 35   72 / 47 / 37   73 / 50 / 38    77 / 58 / 40   139 / 83 / 46   189 / 123 / 76
//   256 x 256      81 / 52 / 42   92 / 58 / 45   93 / 60 / 46   100 / 68 / 49   113 / 80 / 56   203 / 120 / 63
// Above 104 rows, from where 128 x 256 keeps its weights in the caches, the large tiles differ by how they fill the
// CUs: rounds of 256 workgroups of 256 x 256 or of 128 x 256, or 512 of 128 x 128, that take about 8, 5.5 and 5.8
// parts of time (5.4 where 128 x 128 has a CU for each), counted over the tiles that random routing makes.
// 256 x 256 is not taken below 144 workgroups, 128 x 256 below 128, and 128 x 128 where those of 32 x 64 are at
// most two on a CU.  In us, 256 x 256 / 128 x 256 / 128 x 128: 8 experts of [4096, 4096] at 256 rows 60 / 72 /
// -, 160 of [160, 1024] at 160 18.5 / 25.7 / 23.6, 100 of [256, 2048] at 160 26.9 / 20.1 / 24.5, 160 of [384, 1024] at
// 160 37.4 / 40.0 / 31.2, 194 of [373, 888] at 306 84 / - / 54.5; 8 of [4096, 4096] at 106 55.0 / 45.1 / 39.8, 16 of
// [2048, 2048] 23.4 / 17.5 / 18.3, and at 116, where some have two tiles, 24.9 / 17.9 / 23.0; 32 x 64 against 128 x 128:
// 8 of [768, 4096] at 132, 440 workgroups of 32 x 64, 19.9 / 24.1, at 160, 528, 26.1 / 20.6; 1 of [5120, 4096] at 192,
// 480, 20.8 / 20.6, at 224, 560, 25.9 / 21.0; 1 of [4096, 4096] at 256, 512, 20.1 / 21.1.
// Below, 256 columns need more than 128 (256 experts of [64, 4096] at 64 rows: 128 x 128 23.9, 128 x 256 33.3; of
// [128, 4096] 37.1 and 39.0), and a workgroup a CU should not take a round more than 128 x 128's two
// (100 experts of [640, 2048] at 64 rows, 300 workgroups of 128 x 256: 41.3, 128 x 128 30.8).
// Where even 16 x 16 leave little work, they are best whatever the rows (2 experts of [95, 6798] at 111 rows
// 10.9, 32 x 64 17.3; 5 of [46, 4040] at 184 8.2 and 12.7; but 500 workgroups at 20 rows 10.5 and 9.3).
// The host does not know how uneven the routing is.  Where 128 x 256 costs little on an even one, because there
// are many workgroups, it is taken from 4 rows on: 2048 rows over 256 experts of [2048, 7168] take 577 us
// instead of 559 if they are even, but 125 instead of 187 if a few experts have most.  With 512
// workgroups it would lose either way (64 experts of [2048, 4096] at 8 rows: even 125 and 106, uneven 41
// and 41).
// Of the tiles of 32 rows, 512 workgroups of 128 columns run at once, or 768 of 64, in about 4 to 3 parts
// of time: the sums of those rounds decide for short rows (4 rows of each of E experts of [2048, 2048],
// 32 x 64 / 32 x 128: E = 24 19.6 / 20.7 us, 32 29.9 / 24.4, 48 38.0 / 39.5, 64 49.8 / 45.3).  Long rows
// blur the rounds and 64 columns are as good or better (K = 7168: 24 55.9 / 60.4, 48 108 / 108, 96 204 /
// 205; 256 rows over 64 experts, K = 4096: 105 / 110) but where 128 end in a single round and 64 do not
// (32: 78 / 72; at one row each, with experts that got none, 52 / 57).
// Weights that one tile of rows reads (few rows per expert) pass the caches: 32 experts at 48 rows 77
// us, kept in them 88; with several tiles of rows they are shared through L2 (346 rows: 15.5 against
// 17.7 us).
enum Variant { kFew = 16016, k32x64 = 32064, k32x128 = 32128, k128x128 = 128128, k128x256 = 128256, k256x256 = 256256 };
// Rows of an expert up to which one tile of 128 reads its weights, which then pass the caches.
constexpr int64_t kReadOnce = 104;
Variant pick(int64_t rows, int64_t E, int64_t N, int64_t K) {
  const int64_t per = rows / E;
  auto work = [&](int64_t bm, int64_t bn) {
    return ((N + bn - 1) / bn) * std::max(std::min(E, rows), (rows + bm - 1) / bm);
  };
  if (work(16, 16) <= (per <= 16 ? 512 : 400)) return kFew;
  if (per > kReadOnce && N >= 64) {
    // an expert's tiles of bm rows, on the average over random routing: a last one for some of them
    auto tiles = [&](double bm) {
      const double spread = E > 1 ? 2 * std::sqrt((double)per) : 0, least = std::ceil((per - spread) / bm);
      return E * (least + (E > 1 ? std::clamp((per + spread - least * bm) / (2 * spread), 0.0, 1.0) : 0));
    };
    const double g = (double)((N + 255) / 256), t256 = tiles(256) * g, t128 = tiles(128) * g,
                 t64 = tiles(128) * (double)((N + 127) / 128), t32 = tiles(32) * (double)((N + 63) / 64);
    // an average of a hundredth of a round more is no round more yet
    auto rounds = [](double t, double at_once) {
      return t <= 4 * at_once ? std::ceil(t / at_once - 0.01) : t / at_once + 0.5;
    };
    const double c256 = N > 128 && t256 >= 144 ? 8 * rounds(t256, 256) : HUGE_VAL,
                 c128 = N > 128 && t128 >= 128 ? 5.5 * rounds(t128, 256) : HUGE_VAL,
                 c64 = t32 <= 512 ? HUGE_VAL : t64 <= 256 ? 5.4 : 5.8 * rounds(t64, 512);
    if (c256 < HUGE_VAL && c256 <= c128 && c256 <= c64) return k256x256;
    if (c128 < HUGE_VAL && c128 <= c64) return k128x256;
    if (c64 < HUGE_VAL) return k128x128;
  }
  if (N > 128 && per <= kReadOnce) {
    const bool more = (work(128, 256) + 255) / 256 > (work(128, 128) + 511) / 512;
    if (!more && per >= 16 && work(128, 256) >= 140) return k128x256;
    if (!more && per >= 4 && work(128, 256) >= 1024) return k128x256;
  }
  if (per >= 40 && work(128, 128) >= 128) return k128x128;
  const int64_t wide = (work(32, 128) + 511) / 512 * 4, narrow = (work(32, 64) + 767) / 768 * 3;
  if (K < 4096 ? wide <= narrow : rows >= 2 * E && wide == 4 && narrow > 3) return k32x128;
  return k32x64;
}

// Tiles of 256 columns store past the caches, which leaves those to rows and weights: 2048 rows over 32 experts
// of [7168, 2048] 97 us instead of 109, and 113 instead of 124 with the GELU that reads the results; 16
// experts of [2048, 2048] at 128 rows 19.6 and 20.8.  Narrower tiles write parts of lines and lose (13
// experts of [900, 1001] at 128 rows 12.6 and 12.0).  Rows that start inside a line have parts of lines wherever a
// wave's part of a row ends.  16-bit results gain all the same or lose little (346 rows of 32 experts, N = 2047:
// K = 256 33.9 and 32.2, 2048 71.6 and 76.3); fp32 ones of 256 x 256, where a wave writes its columns in two parts,
// one after the other, lose much (52.0 and 33.3, 87.8 and 77.5), and gain where rows start with a line
// (N = 4096: K = 512 67 and 79, 2048 140 and 153).
bool starts_with_lines(const LinearArgs& a, int64_t bytes) {
  return reinterpret_cast<uintptr_t>(a.out) % 128 == 0 && a.out_stride * bytes % 128 == 0;
}

template <typename TO> int launch_linear(const char* who, const LinearArgs& a, hipStream_t s) {
  switch (pick(a.rows, a.E, a.N, a.Kp)) {
    case k256x256:
      if constexpr (ElemInfo<TO>::kBytes == 4)
        if (!starts_with_lines(a, 4))
          return launch_tile<TO, 256, 256, 4, 2, 64, 4, false, kCPolCached, false>(who, a, s);
      return launch_tile<TO, 256, 256, 4, 2, 64, 4, false, kCPolCached>(who, a, s);
    case k128x256:
      if (a.rows / a.E <= kReadOnce) return launch_tile<TO, 128, 256, 2, 4, 128, 3, true, kCPol>(who, a, s);
      return launch_tile<TO, 128, 256, 2, 4, 128, 3, true, kCPolCached>(who, a, s);
    case k128x128: return launch_tile<TO, 128, 128, 2, 2, 64, 4, false, kCPolCached>(who, a, s);
    case k32x128: return launch_tile<TO, 32, 128, 1, 4, 128, 3, true, kCPol>(who, a, s);
    case kFew: return launch_few<TO>(who, a, s);
    default: return launch_tile<TO, 32, 64, 1, 2, 128, 4, true, kCPol>(who, a, s);
  }
}

}  // namespace

extern "C" int64_t fmoe_int8_linear_tile(int64_t rows, int64_t num_experts, int64_t N, int64_t K) {
  if (rows < 1 || num_experts < 1 || N < 1 || K < 1) return -1;
  return pick(rows, num_experts, N, fmoe_host::round_up(K, kRowsPitch));
}

extern "C" int fmoe_int8_linear(const void* d_x, int64_t x_row_stride, int64_t x_rows,
                                const float* d_x_scales, const void* d_index, int index_dtype,
                                const void* d_w, const float* d_w_scales, const void* d_bias,
                                int bias_dtype, const int64_t* d_offsets, int64_t num_experts,
                                int64_t N, int64_t K, int64_t rows, void* d_out,
                                int64_t out_row_stride, int out_dtype, void* stream) {
  fmoe_host::clear_error();
  const char* who = "fmoe_int8_linear";
  FMOE_REQUIRE(rows >= 0 && x_rows >= 0 && N >= 1 && K >= 1 && num_experts >= 1,
               "%s: bad sizes rows=%lld x_rows=%lld N=%lld K=%lld E=%lld", who, (long long)rows,
               (long long)x_rows, (long long)N, (long long)K, (long long)num_experts);
  FMOE_REQUIRE(fmoe_host::is_float_dtype(out_dtype), "%s: bad output dtype %d", who, out_dtype);
  FMOE_REQUIRE(!d_index || fmoe_host::is_index_dtype(index_dtype), "%s: bad index dtype %d", who,
               index_dtype);
  FMOE_REQUIRE(!d_bias || fmoe_host::is_float_dtype(bias_dtype), "%s: bad bias dtype %d", who,
               bias_dtype);
  FMOE_REQUIRE(d_offsets || num_experts == 1, "%s: several experts need row offsets", who);
  FMOE_REQUIRE(out_row_stride >= N, "%s: out row stride %lld is below N=%lld", who,
               (long long)out_row_stride, (long long)N);
  const int64_t Kp = fmoe_host::round_up(K, kRowsPitch);
  FMOE_REQUIRE(x_row_stride % 16 == 0 && x_row_stride >= Kp &&
                   reinterpret_cast<uintptr_t>(d_x) % 16 == 0 &&
                   reinterpret_cast<uintptr_t>(d_w) % 16 == 0,
               "%s: 8-bit rows must start at multiples of 16 bytes and have whole pieces of %d", who,
               kRowsPitch);
  if (K > kMaxK || N > (int64_t(1) << 24) || num_experts > (int64_t(1) << 16) ||
      rows >= (int64_t(1) << 31) || x_rows >= (int64_t(1) << 31)) {
    fmoe_host::set_error("%s: rows=%lld x_rows=%lld N=%lld K=%lld E=%lld too large", who,
                         (long long)rows, (long long)x_rows, (long long)N, (long long)K,
                         (long long)num_experts);
    return FMOE_ERANGE;
  }
  if (rows == 0) return FMOE_OK;
  FMOE_REQUIRE(x_rows >= 1, "%s: rows to write, and none to read", who);
  FMOE_REQUIRE(d_x && d_x_scales && d_w && d_w_scales && d_out, "%s: null device pointer", who);
  const LinearArgs a{static_cast<const uint8_t*>(d_x), x_row_stride, x_rows, d_x_scales, d_index,
                     index_dtype, static_cast<const uint8_t*>(d_w), d_w_scales, d_bias, bias_dtype,
                     d_offsets, num_experts, N, Kp, rows, d_out, out_row_stride, 0};
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (out_dtype == FMOE_F32) return launch_linear<float>(who, a, s);
  if (out_dtype == FMOE_BF16) return launch_linear<bf16_t>(who, a, s);
  return launch_linear<f16_t>(who, a, s);
}
