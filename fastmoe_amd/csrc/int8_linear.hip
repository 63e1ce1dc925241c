// Every expert's product on its own rows, in 8-bit integers:
//
//   out[r, n] = (sum_k x[i(r), k] * w[e(r), n, k]) * sx[i(r)] * sw[e(r), n] + b[e(r), n]
//
// for packed rows r in [off[e], off[e + 1]) of expert e; i(r) = index[r] where the rows are read
// through an index (the dispatch's reverse map: the rows of a token are never copied for its
// experts), else r.  The sums are int32 and exact (K <= 131071 keeps them in range: 128 * 128 * K <
// 2^31), so neither the order nor a split of K changes a bit; each is then converted to fp32 once
// (2^-24), scaled and rounded to the output's type.
//
// Rows and weights lie with K innermost, padded with zeros to whole pieces of 128 bytes, so no
// product needs a tail in K.  Rows of a tile beyond its expert's last repeat that last one, columns
// beyond N repeat the last one; neither is stored.
#include "rows8.h"

#include <algorithm>

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

// A tile of up to BM rows of one expert.  Expert E stands for the rows that belong to none.
struct Tile {
  int64_t expert, row;
  int count;
};

// The `target`-th tile of the packed rows.  Each lane counts one expert's tiles and a prefix sum over
// the wave finds whose the target is; every wave does it for itself, so there is neither a table in
// memory nor a launch that makes it.  Offsets are held to [0, rows]: no value in them makes a wave
// read or write outside the arrays.
template <int BM> __device__ __forceinline__ bool find_tile(const LinearArgs& a, int64_t target, Tile* t) {
  if (!a.off) {
    t->expert = 0;
    t->row = target * BM;
    if (t->row >= a.rows) return false;
    t->count = (int)min((int64_t)BM, a.rows - t->row);
    return true;
  }
  const int lane = threadIdx.x & (kWave - 1);
  int64_t base = 0;
  for (int64_t e0 = 0; e0 <= a.E; e0 += kWave) {
    const int64_t e = e0 + lane;
    int64_t lo = 0, hi = 0;
    if (e <= a.E) {
      lo = e == 0 ? 0 : min(max(a.off[e], (int64_t)0), a.rows);
      hi = e == a.E ? a.rows : min(max(a.off[e + 1], (int64_t)0), a.rows);
    }
    const int n = (int)((max(hi - lo, (int64_t)0) + BM - 1) / BM);
    int incl = n;
#pragma unroll
    for (int d = 1; d < kWave; d *= 2) {
      const int up = __shfl_up(incl, d);
      if (lane >= d) incl += up;
    }
    const int all = __builtin_amdgcn_readlane(incl, kWave - 1);
    if (target < base + all) {
      const int want = (int)(target - base);
      const uint64_t hit = __ballot(want >= incl - n && want < incl);
      const int at = __ffsll((unsigned long long)hit) - 1;
      t->expert = e0 + at;
      const int64_t first = __shfl(lo, at) + (int64_t)(want - __shfl(incl - n, at)) * BM;
      t->row = first;
      t->count = (int)min((int64_t)BM, (int64_t)__shfl(hi, at) - first);
      return true;
    }
    base += all;
  }
  return false;
}

// The row of x that packed row r reads; -1 where its index lies outside x.
__device__ __forceinline__ int64_t source_row(const LinearArgs& a, int64_t r) {
  if (!a.index) return r < a.x_rows ? r : -1;
  const int64_t i = load_index(a.index, a.index_dtype, r);
  return i >= 0 && i < a.x_rows ? i : -1;
}

// Four neighbouring columns of one output row.
template <typename TO>
__device__ __forceinline__ void store4(const LinearArgs& a, const Tile& t, int64_t r, int64_t n,
                                       i32x4 acc, float sx) {
  if (n >= a.N) return;
  TO* p = static_cast<TO*>(a.out) + r * a.out_stride + n;
  float f[4];
  const float* sw = a.sw + t.expert * a.N + n;
  const int left = (int)min((int64_t)4, a.N - n);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    f[i] = 0.f;
    if (i < left) {
      f[i] = (float)acc[i] * sx * sw[i];
      if (a.bias) f[i] += load_weight(a.bias, a.bias_dtype, t.expert * a.N + n + i);
    }
  }
  if (left == 4) {
    if constexpr (ElemInfo<TO>::kBytes == 4)
      *reinterpret_cast<u32x4_any*>(p) = Vec<TO, 4>::pack(f);
    else
      *reinterpret_cast<u32x2_any*>(p) = Vec<TO, 4>::pack(f);
  } else {
    for (int i = 0; i < left; ++i) st1(p + i, f[i]);
  }
}

// Rows of no expert: zeros.
template <typename TO>
__device__ __forceinline__ void zero_rows(const LinearArgs& a, const Tile& t, int64_t n0, int cols) {
  for (int r = 0; r < t.count; ++r)
    for (int64_t n = n0 + threadIdx.x; n < min(n0 + cols, a.N); n += blockDim.x)
      st1(static_cast<TO*>(a.out) + (t.row + r) * a.out_stride + n, 0.f);
}

// Few rows per expert: the weights are the traffic, each byte of them used for at most 16 * MT rows.
// A workgroup has 16 * MT rows and 16 * NB columns of one expert.  Its waves take 128-byte pieces of
// K in turn, straight from memory to the matrix units' registers (LDS would only add a copy: no
// two waves share a byte of the weights), and add their int32 parts in LDS at the end.
template <typename TO, int MT, int NB, int WAVES>
__global__ __launch_bounds__(WAVES * kWave) void k_int8_stream(LinearArgs a) {
  __shared__ i32x4 part[WAVES][MT * NB][kWave];
  Tile t;
  if (!find_tile<16 * MT>(a, blockIdx.x / (unsigned)a.groups_n, &t)) return;
  const int64_t n0 = (int64_t)(blockIdx.x % (unsigned)a.groups_n) * (16 * NB);
  if (t.expert == a.E) {
    zero_rows<TO>(a, t, n0, 16 * NB);
    return;
  }
  const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
  const int l16 = lane & 15, quad = lane >> 4;
  const uint8_t* xp[MT];
#pragma unroll
  for (int m = 0; m < MT; ++m) {
    const int64_t i = source_row(a, t.row + min(m * 16 + l16, t.count - 1));
    xp[m] = a.x + max(i, (int64_t)0) * a.x_stride + quad * 16;
  }
  const uint8_t* wp[NB];
#pragma unroll
  for (int b = 0; b < NB; ++b)
    wp[b] = a.w + (t.expert * a.N + min(n0 + b * 16 + l16, a.N - 1)) * a.Kp + quad * 16;
  i32x4 acc[MT][NB];
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int b = 0; b < NB; ++b) acc[m][b] = i32x4{0, 0, 0, 0};
  for (int64_t k = wave * 128; k < a.Kp; k += WAVES * 128) {
    i32x4 xv[2][MT], wv[2][NB];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
#pragma unroll
      for (int b = 0; b < NB; ++b)
        wv[h][b] = __builtin_nontemporal_load(reinterpret_cast<const i32x4*>(wp[b] + k + 64 * h));
#pragma unroll
      for (int m = 0; m < MT; ++m) xv[h][m] = *reinterpret_cast<const i32x4*>(xp[m] + k + 64 * h);
    }
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int b = 0; b < NB; ++b)
          acc[m][b] = __builtin_amdgcn_mfma_i32_16x16x64_i8(wv[h][b], xv[h][m], acc[m][b], 0, 0, 0);
  }
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int b = 0; b < NB; ++b) part[wave][m * NB + b][lane] = acc[m][b];
  __syncthreads();
  // lane l of a 16 x 16 result has row l % 16 and columns 4 * (l / 16) + 0..3
  for (int p = wave; p < MT * NB; p += WAVES) {
    i32x4 sum = part[0][p][lane];
#pragma unroll
    for (int v = 1; v < WAVES; ++v) sum += part[v][p][lane];
    const int m = (p / NB) * 16 + l16;
    if (m < t.count) {
      const int64_t i = source_row(a, t.row + m);
      store4<TO>(a, t, t.row + m, n0 + (p % NB) * 16 + quad * 4, i >= 0 ? sum : i32x4{0, 0, 0, 0},
                 i >= 0 ? a.sx[i] : 0.f);
    }
  }
}

}  // namespace fmoe

using namespace fmoe;

namespace {

constexpr int64_t kMaxK = 131071;

// Tiles of `bm` rows that `rows` packed rows of up to `E` experts (and of none) have at most.
int64_t most_tiles(int64_t rows, int64_t E, bool grouped, int64_t bm) {
  const int64_t even = (rows + bm - 1) / bm;
  return grouped ? std::min(rows, even + E) : even;
}

template <typename TO, int MT, int NB, int WAVES> int launch_stream(const char* who, LinearArgs a, hipStream_t s) {
  const int64_t tiles = most_tiles(a.rows, a.E, a.off != nullptr, 16 * MT);
  a.groups_n = (int)((a.N + 16 * NB - 1) / (16 * NB));
  if (tiles > ((int64_t(1) << 32) - 1) / (a.groups_n * (int64_t)WAVES * kWave)) {
    fmoe_host::set_error("%s: rows=%lld N=%lld too large", who, (long long)a.rows, (long long)a.N);
    return FMOE_ERANGE;
  }
  hipLaunchKernelGGL((k_int8_stream<TO, MT, NB, WAVES>), dim3((unsigned)(tiles * a.groups_n)),
                     dim3(WAVES * kWave), 0, s, a);
  return fmoe_host::check_launch(who);
}

template <typename TO> int launch_linear(const char* who, const LinearArgs& a, hipStream_t s) {
  return launch_stream<TO, 4, 4, 4>(who, a, s);
}

}  // namespace

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
