// Root-mean-square norm with the residual's addition (forward, backward, 8-bit rows), and rows to
// 8 bits and back.
//
//   h = x + residual, rounded to x's type: the residual stream as it is stored
//   c = 1 / sqrt(mean(h^2) + eps);  y = h * c * w, in fp32, rounded once
//   8 bits: s = max|y| / 127, q = rint(y * (127 / max|y|)) of the fp32 y
//
//   backward, with t = grad_y * w:
//   grad_x = grad_residual = grad_h + c * t - h * c^3 / D * sum(t * h)
//   grad_w = sum over rows of grad_y * h * c
//
// Sums, the norm's factor and the scales are fp32; a row whose sum of squares passes fp32's range (finite
// values of 1.5e17 in 16384 columns, 1.5e18 in 150) gives zeros, as it does in the unfused fp32 formula.
#include "rows8.h"

#include <algorithm>

namespace fmoe {

// A row is held in registers by THREADS threads, VPT vectors of eight columns each, so every
// input is read from HBM once and both reductions (the squares' sum, then the largest |y|) run on
// registers.  THREADS == 64 puts four rows in a workgroup, without any barrier.
template <int THREADS> constexpr int rows_per_group() { return THREADS < kGroup ? kGroup / THREADS : 1; }
template <int THREADS> constexpr int group_threads() { return THREADS < kGroup ? kGroup : THREADS; }

struct NormArgs {
  const void *x, *residual, *weight;
  int64_t x_stride, r_stride;  // elements
  int64_t rows, cols;
  float eps;
  void *h, *y;    // packed; null where not wanted
  int stream_y;   // store y past the caches
  float* rstd;    // null where not wanted
  uint8_t* q;     // null where not wanted
  int64_t q_stride, q_cols;  // bytes from row to row; bytes written of each: the columns, zeros after them
  float* scales;
};

template <typename T, typename TW, int THREADS, int VPT>
__global__ __launch_bounds__(group_threads<THREADS>()) void k_norm(NormArgs a) {
  __shared__ float lds_sum[16];
  __shared__ uint32_t lds_max[16];
  constexpr int kRows = rows_per_group<THREADS>();
  const int64_t row = (int64_t)blockIdx.x * kRows + threadIdx.x / THREADS;
  if (row >= a.rows) return;  // whole waves (THREADS == 64) or the whole workgroup
  const int tid = threadIdx.x % THREADS;
  using V = Eight<T>;
  using W = Eight<TW>;
  const T* x = static_cast<const T*>(a.x) + row * a.x_stride;
  typename V::raw_t xr[VPT], rr[VPT];
  typename W::raw_t wr[VPT];
#pragma unroll
  for (int v = 0; v < VPT; ++v) xr[v] = V::template load<true>(x, (v * THREADS + tid) * 8, a.cols);
  if (a.residual) {
    const T* r = static_cast<const T*>(a.residual) + row * a.r_stride;
#pragma unroll
    for (int v = 0; v < VPT; ++v) rr[v] = V::template load<true>(r, (v * THREADS + tid) * 8, a.cols);
  }
#pragma unroll
  for (int v = 0; v < VPT; ++v)
    wr[v] = W::template load<false>(static_cast<const TW*>(a.weight), (v * THREADS + tid) * 8, a.cols);

  float f[VPT][8];
  float sum = 0.f;
#pragma unroll
  for (int v = 0; v < VPT; ++v) {
    V::V::cvt(xr[v], f[v]);
    if (a.residual) {
      float r[8];
      V::V::cvt(rr[v], r);
#pragma unroll
      for (int i = 0; i < 8; ++i) f[v][i] += r[i];
      const typename V::raw_t h = V::V::pack(f[v]);
      V::store(static_cast<T*>(a.h) + row * a.cols, (v * THREADS + tid) * 8, a.cols, h);
      V::V::cvt(h, f[v]);  // the stream is normalised as it is stored
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) sum = __builtin_fmaf(f[v][i], f[v][i], sum);
  }
  const float c = 1.0f / sqrtf(group_sum<THREADS>(sum, lds_sum) / (float)a.cols + a.eps);
  if (a.rstd && tid == 0) a.rstd[row] = c;
  float top = 0.f;
#pragma unroll
  for (int v = 0; v < VPT; ++v) {
    float w[8];
    W::V::cvt(wr[v], w);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      f[v][i] = f[v][i] * c * w[i];
      top = larger(top, f[v][i]);
    }
    if (a.y) {
      T* y = static_cast<T*>(a.y) + row * a.cols;
      const typename V::raw_t p = V::V::pack(f[v]);
      if (a.stream_y) V::template store<true>(y, (v * THREADS + tid) * 8, a.cols, p);
      else V::store(y, (v * THREADS + tid) * 8, a.cols, p);
    }
  }
  if (!a.q) return;
  const Scale8 s = scale8(group_max<THREADS>(abs_bits(top), lds_max));
  if (tid == 0) a.scales[row] = s.scale;
  uint8_t* q = a.q + row * a.q_stride;
#pragma unroll
  for (int v = 0; v < VPT; ++v) {
    const int col = (v * THREADS + tid) * 8;
    if (col < a.q_cols) *reinterpret_cast<u32x2*>(q + col) = pack8(f[v], s);
  }
}

// Rows longer than the registers hold: the same steps, each over the row again.  A thread reads back
// only what it wrote or read itself.
template <typename T, typename TW>
__global__ __launch_bounds__(1024) void k_norm_long(NormArgs a) {
  __shared__ float lds_sum[16];
  __shared__ uint32_t lds_max[16];
  constexpr int kThreads = 1024;
  const int64_t row = blockIdx.x;
  using V = Eight<T>;
  using W = Eight<TW>;
  const T* x = static_cast<const T*>(a.x) + row * a.x_stride;
  const T* r = a.residual ? static_cast<const T*>(a.residual) + row * a.r_stride : nullptr;
  T* h = r ? static_cast<T*>(a.h) + row * a.cols : nullptr;
  const T* in = r ? h : x;
  float sum = 0.f;
  for (int64_t col = threadIdx.x * 8; col < a.cols; col += kThreads * 8) {
    float f[8];
    V::V::cvt(V::template load<false>(x, col, a.cols), f);
    if (r) {
      float g[8];
      V::V::cvt(V::template load<false>(r, col, a.cols), g);
#pragma unroll
      for (int i = 0; i < 8; ++i) f[i] += g[i];
      const typename V::raw_t p = V::V::pack(f);
      V::store(h, col, a.cols, p);
      V::V::cvt(p, f);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) sum = __builtin_fmaf(f[i], f[i], sum);
  }
  const float c = 1.0f / sqrtf(group_sum<kThreads>(sum, lds_sum) / (float)a.cols + a.eps);
  if (a.rstd && threadIdx.x == 0) a.rstd[row] = c;
  auto normed = [&](int64_t col, float* f) {
    float w[8];
    V::V::cvt(V::template load<false>(in, col, a.cols), f);
    W::V::cvt(W::template load<false>(static_cast<const TW*>(a.weight), col, a.cols), w);
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = f[i] * c * w[i];
  };
  float top = 0.f;
  for (int64_t col = threadIdx.x * 8; col < a.cols; col += kThreads * 8) {
    float f[8];
    normed(col, f);
#pragma unroll
    for (int i = 0; i < 8; ++i) top = larger(top, f[i]);
    if (a.y) V::store(static_cast<T*>(a.y) + row * a.cols, col, a.cols, V::V::pack(f));
  }
  if (!a.q) return;
  const Scale8 s = scale8(group_max<kThreads>(abs_bits(top), lds_max));
  if (threadIdx.x == 0) a.scales[row] = s.scale;
  for (int64_t col = threadIdx.x * 8; col < a.q_cols; col += kThreads * 8) {
    float f[8];
    normed(col, f);
    *reinterpret_cast<u32x2*>(a.q + row * a.q_stride + col) = pack8(f, s);
  }
}

struct NormBwdArgs {
  const void *gy, *gh, *h, *weight;  // gh null: no gradient comes through the stream
  const float* rstd;
  int64_t gy_stride, gh_stride, h_stride;  // elements
  int64_t rows, cols;
  void* gx;         // packed
  float* partials;  // [workgroups, cols]: each one's sum over its rows of grad_y * h * c; or null
  int64_t units;    // rows in flight: workgroups times rows_per_group
};

// A unit (the threads that hold a row) takes rows unit, unit + units, ... and keeps its part of
// grad_w in registers: one pass over the three inputs, whatever the number of rows.  Where a unit is a
// wave, the workgroup's four join their parts in LDS.
template <typename T, typename TW, int THREADS, int VPT>
__global__ __launch_bounds__(group_threads<THREADS>()) void k_norm_bwd(NormBwdArgs a) {
  __shared__ float lds[2][16];
  constexpr int kRows = rows_per_group<THREADS>();
  __shared__ float join[kRows > 1 ? kRows : 1][kRows > 1 ? THREADS * VPT * 8 : 1];
  const int64_t unit = (int64_t)blockIdx.x * kRows + threadIdx.x / THREADS;
  const int tid = threadIdx.x % THREADS;
  using V = Eight<T>;
  using W = Eight<TW>;
  float w[VPT][8], gw[VPT][8];
#pragma unroll
  for (int v = 0; v < VPT; ++v) {
    W::V::cvt(W::template load<false>(static_cast<const TW*>(a.weight), (v * THREADS + tid) * 8,
                                      a.cols), w[v]);
#pragma unroll
    for (int i = 0; i < 8; ++i) gw[v][i] = 0.f;
  }
  const float inv_cols = 1.0f / (float)a.cols;
  struct Row {
    typename V::raw_t gy[VPT], h[VPT], gh[VPT];
    float c;
  };
  auto load = [&](int64_t row, Row& r) {
    const T* gyp = static_cast<const T*>(a.gy) + row * a.gy_stride;
    const T* hp = static_cast<const T*>(a.h) + row * a.h_stride;
#pragma unroll
    for (int v = 0; v < VPT; ++v) {
      r.gy[v] = V::template load<true>(gyp, (v * THREADS + tid) * 8, a.cols);
      r.h[v] = V::template load<true>(hp, (v * THREADS + tid) * 8, a.cols);
    }
    if (a.gh) {
      const T* ghp = static_cast<const T*>(a.gh) + row * a.gh_stride;
#pragma unroll
      for (int v = 0; v < VPT; ++v)
        r.gh[v] = V::template load<true>(ghp, (v * THREADS + tid) * 8, a.cols);
    } else {
#pragma unroll
      for (int v = 0; v < VPT; ++v) r.gh[v] = V::zero();
    }
    r.c = a.rstd[row];
  };
  // The next row is asked for before this one's sum is joined, where the registers hold both.
  constexpr bool kAhead = ElemInfo<T>::kBytes == 2 && THREADS <= 512;
  Row now, next;
  if (kAhead && unit < a.rows) load(unit, now);
  int turn = 0;
  for (int64_t row = unit; row < a.rows; row += a.units, turn ^= 1) {
    if constexpr (!kAhead) load(row, now);
    else if (row + a.units < a.rows) load(row + a.units, next);
    float sum = 0.f;
#pragma unroll
    for (int v = 0; v < VPT; ++v) {
      float g[8], f[8];
      V::V::cvt(now.gy[v], g);
      V::V::cvt(now.h[v], f);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float hat = f[i] * now.c;
        gw[v][i] = __builtin_fmaf(g[i], hat, gw[v][i]);
        sum = __builtin_fmaf(g[i] * w[v][i], hat, sum);
      }
    }
    // two words of LDS per wave, used in turn: a thread that is a row ahead writes the other
    const float m = group_sum<THREADS>(sum, lds[turn]) * inv_cols;
    T* gx = static_cast<T*>(a.gx) + row * a.cols;
#pragma unroll
    for (int v = 0; v < VPT; ++v) {
      float g[8], f[8], r[8];
      V::V::cvt(now.gy[v], g);
      V::V::cvt(now.h[v], f);
      V::V::cvt(now.gh[v], r);
#pragma unroll
      for (int i = 0; i < 8; ++i)
        r[i] = __builtin_fmaf(now.c, __builtin_fmaf(-(f[i] * now.c), m, g[i] * w[v][i]), r[i]);
      V::store(gx, (v * THREADS + tid) * 8, a.cols, V::V::pack(r));
    }
    if constexpr (kAhead) now = next;
  }
  if (!a.partials) return;
  float* out = a.partials + (int64_t)blockIdx.x * a.cols;
  if constexpr (kRows > 1) {
    float* mine = join[threadIdx.x / THREADS];
#pragma unroll
    for (int v = 0; v < VPT; ++v)
#pragma unroll
      for (int i = 0; i < 8; ++i) mine[(v * 8 + i) * THREADS + tid] = gw[v][i];
    __syncthreads();
    if (threadIdx.x >= THREADS) return;
#pragma unroll
    for (int v = 0; v < VPT; ++v)
#pragma unroll
      for (int i = 0; i < 8; ++i)
#pragma unroll
        for (int r = 1; r < kRows; ++r) gw[v][i] += join[r][(v * 8 + i) * THREADS + tid];
  }
#pragma unroll
  for (int v = 0; v < VPT; ++v) {
    const int64_t col = (v * THREADS + tid) * 8;
    Eight<float>::store(out, col, a.cols, Eight<float>::V::pack(gw[v]));
  }
}

// Rows longer than the registers hold: grad_x row by row, grad_w's parts column by column.
template <typename T, typename TW>
__global__ __launch_bounds__(1024) void k_norm_bwd_long(NormBwdArgs a) {
  __shared__ float lds[16];
  constexpr int kThreads = 1024;
  const int64_t row = blockIdx.x;
  using V = Eight<T>;
  using W = Eight<TW>;
  const T* gyp = static_cast<const T*>(a.gy) + row * a.gy_stride;
  const T* hp = static_cast<const T*>(a.h) + row * a.h_stride;
  const T* ghp = a.gh ? static_cast<const T*>(a.gh) + row * a.gh_stride : nullptr;
  const float c = a.rstd[row];
  float g[8], f[8], w[8];
  auto read = [&](int64_t col) {
    V::V::cvt(V::template load<false>(gyp, col, a.cols), g);
    V::V::cvt(V::template load<false>(hp, col, a.cols), f);
    W::V::cvt(W::template load<false>(static_cast<const TW*>(a.weight), col, a.cols), w);
  };
  float sum = 0.f;
  for (int64_t col = threadIdx.x * 8; col < a.cols; col += kThreads * 8) {
    read(col);
#pragma unroll
    for (int i = 0; i < 8; ++i) sum = __builtin_fmaf(g[i] * w[i], f[i] * c, sum);
  }
  const float m = group_sum<kThreads>(sum, lds) * (1.0f / (float)a.cols);
  for (int64_t col = threadIdx.x * 8; col < a.cols; col += kThreads * 8) {
    float r[8];
    read(col);
    V::V::cvt(ghp ? V::template load<false>(ghp, col, a.cols) : V::zero(), r);
#pragma unroll
    for (int i = 0; i < 8; ++i)
      r[i] = __builtin_fmaf(c, __builtin_fmaf(-(f[i] * c), m, g[i] * w[i]), r[i]);
    V::store(static_cast<T*>(a.gx) + row * a.cols, col, a.cols, V::V::pack(r));
  }
}

template <typename T>
__global__ __launch_bounds__(kGroup) void k_norm_bwd_long_w(NormBwdArgs a) {
  using V = Eight<T>;
  const int64_t unit = blockIdx.x;
  const int64_t col = ((int64_t)blockIdx.y * kGroup + threadIdx.x) * 8;
  if (col >= a.cols) return;
  float gw[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  for (int64_t row = unit; row < a.rows; row += a.units) {
    float g[8], f[8];
    V::V::cvt(V::template load<false>(static_cast<const T*>(a.gy) + row * a.gy_stride, col, a.cols), g);
    V::V::cvt(V::template load<false>(static_cast<const T*>(a.h) + row * a.h_stride, col, a.cols), f);
    const float c = a.rstd[row];
#pragma unroll
    for (int i = 0; i < 8; ++i) gw[i] = __builtin_fmaf(g[i], f[i] * c, gw[i]);
  }
  Eight<float>::store(a.partials + unit * a.cols, col, a.cols, Eight<float>::V::pack(gw));
}

// grad_w[c] = sum over the parts of partials[part, c], each column in one fixed order: a workgroup takes 64
// columns, its sixteen waves every sixteenth part.  (Four waves took 7.7 us for 512 parts of 16384.)
constexpr int kSumWaves = 16;
template <typename TW>
__global__ __launch_bounds__(kSumWaves * kWave) void k_norm_bwd_w(const float* __restrict__ partials,
                                                                  int64_t parts, int64_t cols,
                                                                  TW* __restrict__ out) {
  __shared__ float lds[kSumWaves][kWave];
  const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
  const int64_t col = (int64_t)blockIdx.x * kWave + lane;
  float sum = 0.f;
  if (col < cols) {
#pragma unroll 8
    for (int64_t p = wave; p < parts; p += kSumWaves) sum += partials[p * cols + col];
  }
  lds[wave][lane] = sum;
  __syncthreads();
  if (wave == 0 && col < cols) {
#pragma unroll
    for (int v = 1; v < kSumWaves; ++v) sum += lds[v][lane];
    st1(out + col, sum);
  }
}

// ---- rows to 8 bits and back ----------------------------------------------------------------
struct RowsArgs {
  const void* x;
  int64_t x_stride, rows, cols;
  uint8_t* q;
  int64_t q_stride, q_cols;  // bytes from row to row; bytes written of each: the columns, zeros after them
  float* scales;
};

template <typename T, bool GELU, int THREADS, int VPT>
__global__ __launch_bounds__(group_threads<THREADS>()) void k_rows8(RowsArgs a) {
  __shared__ uint32_t lds[16];
  constexpr int kRows = rows_per_group<THREADS>();
  const int64_t row = (int64_t)blockIdx.x * kRows + threadIdx.x / THREADS;
  if (row >= a.rows) return;
  const int tid = threadIdx.x % THREADS;
  using V = Eight<T>;
  const T* x = static_cast<const T*>(a.x) + row * a.x_stride;
  typename V::raw_t raw[VPT];
#pragma unroll
  for (int v = 0; v < VPT; ++v) raw[v] = V::template load<true>(x, (v * THREADS + tid) * 8, a.cols);
  float f[VPT][8];
  float top = 0.f;
#pragma unroll
  for (int v = 0; v < VPT; ++v) {
    V::V::cvt(raw[v], f[v]);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if constexpr (GELU) f[v][i] = gelu8<T>(f[v][i]);
      top = larger(top, f[v][i]);
    }
  }
  const Scale8 s = scale8(group_max<THREADS>(abs_bits(top), lds));
  if (tid == 0) a.scales[row] = s.scale;
  uint8_t* q = a.q + row * a.q_stride;
#pragma unroll
  for (int v = 0; v < VPT; ++v) {
    const int col = (v * THREADS + tid) * 8;
    if (col < a.q_cols) *reinterpret_cast<u32x2*>(q + col) = pack8(f[v], s);
  }
}

template <typename T, bool GELU>
__global__ __launch_bounds__(1024) void k_rows8_long(RowsArgs a) {
  __shared__ uint32_t lds[16];
  constexpr int kThreads = 1024;
  const int64_t row = blockIdx.x;
  using V = Eight<T>;
  const T* x = static_cast<const T*>(a.x) + row * a.x_stride;
  auto read = [&](int64_t col, float* f) {
    V::V::cvt(V::template load<false>(x, col, a.cols), f);
    if constexpr (GELU) {
#pragma unroll
      for (int i = 0; i < 8; ++i) f[i] = gelu8<T>(f[i]);
    }
  };
  float top = 0.f;
  for (int64_t col = threadIdx.x * 8; col < a.cols; col += kThreads * 8) {
    float f[8];
    read(col, f);
#pragma unroll
    for (int i = 0; i < 8; ++i) top = larger(top, f[i]);
  }
  const Scale8 s = scale8(group_max<kThreads>(abs_bits(top), lds));
  if (threadIdx.x == 0) a.scales[row] = s.scale;
  for (int64_t col = threadIdx.x * 8; col < a.q_cols; col += kThreads * 8) {
    float f[8];
    read(col, f);
    *reinterpret_cast<u32x2*>(a.q + row * a.q_stride + col) = pack8(f, s);
  }
}

}  // namespace fmoe

using namespace fmoe;

namespace {

constexpr int kMaxRegCols = 16384;          // columns that the largest register variant holds
// Workgroups of the backward, as many parts of grad_w.  The large ones fill a CU: one for each (2048 x 7168:
// 27 us, 31 with two; smaller ones 42 us with two at 16384 x 2048, 58 with one).
constexpr int64_t kBwdGroups = 512;
template <int THREADS> constexpr int64_t bwd_groups() { return THREADS >= 512 ? kBwdGroups / 2 : kBwdGroups; }
// y is stored past the caches from the size at which the combine's output is: 4096 x 16384 takes 83
// instead of 95 us.  (8192 x 4096, 64 MiB, takes 47 either way, and leaves y to its reader in the cache.)
int streams_y(int64_t bytes) { return bytes >= FMOE_STREAM_OUT_BYTES; }
constexpr int64_t kMaxCols = int64_t(1) << 26;  // 2048 columns for each of a grid's 2^15 in y

// Calls f(threads, vectors) with the variant that holds a row of `cols` in at most four vectors a thread.
// Up to 2048 columns a row is a wave's: no barrier, and more of its loads in flight (GELU to 8 bits of
// 49152 x 2048: 64 us against 77 with 256 threads; the norm 46 against 48).  At 4096 columns 256
// threads are better than 512 (43 against 51 us), beyond that there is little between them.
template <typename F> void by_cols(int64_t cols, F&& f) {
  using std::integral_constant;
  const int64_t v = (cols + 7) / 8;
  auto go = [&](auto t, auto n) { f(t, n); };
  if (v <= 64) go(integral_constant<int, 64>{}, integral_constant<int, 1>{});
  else if (v <= 128) go(integral_constant<int, 64>{}, integral_constant<int, 2>{});
  else if (v <= 256) go(integral_constant<int, 64>{}, integral_constant<int, 4>{});
  else if (v <= 512) go(integral_constant<int, 256>{}, integral_constant<int, 2>{});
  else if (v <= 1024) go(integral_constant<int, 256>{}, integral_constant<int, 4>{});
  else go(integral_constant<int, 512>{}, integral_constant<int, 4>{});
}
// The backward holds three inputs, the weight and its gradient's part: two vectors each (four take 250
// registers).  Above 8192 columns none fits: with 1024 threads and two vectors 16-bit rows spill 5 registers (23
// with an fp32 weight), fp32 rows 55, and 53 with 512 and four, which they take.
template <typename T, typename F> void by_cols_backward(int64_t cols, F&& f) {
  using std::integral_constant;
  const int64_t v = (cols + 7) / 8;
  auto go = [&](auto t, auto n) { f(t, n); };
  if (v <= 64) go(integral_constant<int, 64>{}, integral_constant<int, 1>{});
  else if (v <= 128) go(integral_constant<int, 64>{}, integral_constant<int, 2>{});
  else if (v <= 256) go(integral_constant<int, 256>{}, integral_constant<int, 1>{});
  else if (v <= 512) go(integral_constant<int, 256>{}, integral_constant<int, 2>{});
  else if (v <= 1024) go(integral_constant<int, 512>{}, integral_constant<int, 2>{});
  else if constexpr (std::is_same<T, float>::value) go(integral_constant<int, 512>{}, integral_constant<int, 4>{});
  else go(integral_constant<int, 1024>{}, integral_constant<int, 2>{});
}

template <typename F> void by_float(int dtype, F&& f) {
  if (dtype == FMOE_F32) f(float{});
  else if (dtype == FMOE_BF16) f(bf16_t{});
  else f(f16_t{});
}

// The weight has the rows' type or fp32.
template <typename F> void by_weight(int dtype, int w_dtype, F&& f) {
  by_float(dtype, [&](auto t) {
    if (w_dtype == dtype) f(t, t);
    else f(t, float{});
  });
}

int check_sizes(const char* who, int64_t rows, int64_t cols, int dtype) {
  FMOE_REQUIRE(rows >= 0 && cols >= 1, "%s: bad sizes rows=%lld columns=%lld", who, (long long)rows,
               (long long)cols);
  FMOE_REQUIRE(fmoe_host::is_float_dtype(dtype), "%s: bad dtype %d", who, dtype);
  // a launch has fewer than 2^32 threads: by_cols's for each row, and a workgroup to spare
  const int64_t threads = cols <= 2048 ? 64 : cols <= 8192 ? 256 : 1024;
  if (cols > kMaxCols || rows > ((int64_t(1) << 32) - 1024) / threads) {
    fmoe_host::set_error("%s: rows=%lld or columns=%lld too large", who, (long long)rows,
                         (long long)cols);
    return FMOE_ERANGE;
  }
  return FMOE_OK;
}

int check_rows8(const char* who, const void* q, int64_t q_stride, const void* scales, int64_t rows,
                int64_t cols) {
  FMOE_REQUIRE(rows == 0 || (q && scales), "%s: null device pointer", who);
  FMOE_REQUIRE(reinterpret_cast<uintptr_t>(q) % 16 == 0 && q_stride % 16 == 0,
               "%s: 8-bit rows must start at multiples of 16 bytes", who);
  FMOE_REQUIRE(q_stride >= fmoe_host::round_up(cols, kRowsPitch),
               "%s: 8-bit row pitch %lld is below %lld columns in whole pieces of %d", who,
               (long long)q_stride, (long long)cols, kRowsPitch);
  return FMOE_OK;
}

int check_norm_weight(const char* who, const void* w, int w_dtype, int dtype) {
  FMOE_REQUIRE(w, "%s: null device pointer", who);
  FMOE_REQUIRE(w_dtype == dtype || w_dtype == FMOE_F32,
               "%s: the weight must have the rows' dtype or fp32", who);
  return FMOE_OK;
}

template <int THREADS> dim3 row_grid(int64_t rows) {
  constexpr int per = rows_per_group<THREADS>();
  return dim3((unsigned)((rows + per - 1) / per));
}

}  // namespace

extern "C" int fmoe_add_rms_norm(const void* d_x, int64_t x_row_stride, const void* d_residual,
                                 int64_t residual_row_stride, const void* d_weight, int weight_dtype,
                                 int64_t rows, int64_t cols, int dtype, float eps, void* d_h,
                                 void* d_y, float* d_rstd, void* d_q, int64_t q_stride,
                                 float* d_scales, void* stream) {
  fmoe_host::clear_error();
  const char* who = "fmoe_add_rms_norm";
  if (int rc = check_sizes(who, rows, cols, dtype)) return rc;
  if (int rc = check_norm_weight(who, d_weight, weight_dtype, dtype)) return rc;
  FMOE_REQUIRE(rows == 0 || d_x, "%s: null device pointer", who);
  FMOE_REQUIRE(!d_residual || d_h || rows == 0, "%s: a residual needs the stream's output", who);
  FMOE_REQUIRE(x_row_stride >= 0 && residual_row_stride >= 0, "%s: negative row stride", who);
  if (d_q || q_stride)
    if (int rc = check_rows8(who, d_q, q_stride, d_scales, rows, cols)) return rc;
  if (rows == 0) return FMOE_OK;
  const NormArgs a{d_x, d_residual, d_weight, x_row_stride, residual_row_stride, rows, cols, eps,
                   d_h, d_y, streams_y(rows * cols * fmoe_host::dtype_bytes(dtype)), d_rstd,
                   static_cast<uint8_t*>(d_q), q_stride,
                   fmoe_host::round_up(cols, kRowsPitch), d_scales};
  hipStream_t s = static_cast<hipStream_t>(stream);
  by_weight(dtype, weight_dtype, [&](auto t, auto tw) {
    using T = decltype(t);
    using TW = decltype(tw);
    if (cols > kMaxRegCols) {
      hipLaunchKernelGGL((k_norm_long<T, TW>), dim3((unsigned)rows), dim3(1024), 0, s, a);
      return;
    }
    by_cols(cols, [&](auto th, auto v) {
      constexpr int kT = decltype(th)::value;
      hipLaunchKernelGGL((k_norm<T, TW, kT, decltype(v)::value>), row_grid<kT>(rows),
                         dim3(group_threads<kT>()), 0, s, a);
    });
  });
  return fmoe_host::check_launch(who);
}

extern "C" int64_t fmoe_add_rms_norm_backward_workspace_bytes(int64_t rows, int64_t cols) {
  if (rows < 0 || cols < 1) return -1;
  return std::max<int64_t>(std::min(rows, kBwdGroups), 1) * cols * 4;
}

extern "C" int fmoe_add_rms_norm_backward(const void* d_grad_y, int64_t gy_row_stride,
                                          const void* d_grad_h, int64_t gh_row_stride,
                                          const void* d_h, int64_t h_row_stride,
                                          const void* d_weight, int weight_dtype,
                                          const float* d_rstd, int64_t rows, int64_t cols,
                                          int dtype, void* d_grad_x, void* d_grad_w,
                                          void* d_workspace, int64_t workspace_bytes,
                                          void* stream) {
  fmoe_host::clear_error();
  const char* who = "fmoe_add_rms_norm_backward";
  if (int rc = check_sizes(who, rows, cols, dtype)) return rc;
  if (int rc = check_norm_weight(who, d_weight, weight_dtype, dtype)) return rc;
  FMOE_REQUIRE(rows == 0 || (d_grad_y && d_h && d_rstd && d_grad_x), "%s: null device pointer", who);
  FMOE_REQUIRE(gy_row_stride >= 0 && gh_row_stride >= 0 && h_row_stride >= 0,
               "%s: negative row stride", who);
  const int64_t need = fmoe_add_rms_norm_backward_workspace_bytes(rows, cols);
  FMOE_REQUIRE(!d_grad_w || (d_workspace && workspace_bytes >= need &&
                             reinterpret_cast<uintptr_t>(d_workspace) % 16 == 0),
               "%s: the weight's gradient needs an aligned workspace of %lld bytes", who,
               (long long)need);
  NormBwdArgs a{d_grad_y, d_grad_h, d_h, d_weight, d_rstd, gy_row_stride, gh_row_stride,
                h_row_stride, rows, cols, d_grad_x,
                d_grad_w ? static_cast<float*>(d_workspace) : nullptr, 0};
  hipStream_t s = static_cast<hipStream_t>(stream);
  int64_t parts = 0;
  if (rows > 0) {
    by_weight(dtype, weight_dtype, [&](auto t, auto tw) {
      using T = decltype(t);
      using TW = decltype(tw);
      if (cols > kMaxRegCols) {
        a.units = parts = std::min(rows, kBwdGroups);
        hipLaunchKernelGGL((k_norm_bwd_long<T, TW>), dim3((unsigned)rows), dim3(1024), 0, s, a);
        if (d_grad_w)
          hipLaunchKernelGGL((k_norm_bwd_long_w<T>),
                             dim3((unsigned)parts, (unsigned)((cols + kGroup * 8 - 1) / (kGroup * 8))),
                             dim3(kGroup), 0, s, a);
        return;
      }
      by_cols_backward<T>(cols, [&](auto th, auto v) {
        constexpr int kT = decltype(th)::value, kRows = rows_per_group<kT>();
        parts = std::min((rows + kRows - 1) / kRows, bwd_groups<kT>());
        a.units = parts * kRows;
        hipLaunchKernelGGL((k_norm_bwd<T, TW, kT, decltype(v)::value>), dim3((unsigned)parts),
                           dim3(group_threads<kT>()), 0, s, a);
      });
    });
  }
  if (d_grad_w)
    by_float(weight_dtype, [&](auto tw) {
      using TW = decltype(tw);
      hipLaunchKernelGGL((k_norm_bwd_w<TW>), dim3((unsigned)((cols + kWave - 1) / kWave)),
                         dim3(kSumWaves * kWave), 0, s, a.partials, parts, cols,
                         static_cast<TW*>(d_grad_w));
    });
  return fmoe_host::check_launch(who);
}

extern "C" int fmoe_quantize_rows(const void* d_x, int64_t x_row_stride, int64_t rows, int64_t cols,
                                  int dtype, int activation, void* d_q, int64_t q_stride,
                                  float* d_scales, void* stream) {
  fmoe_host::clear_error();
  const char* who = "fmoe_quantize_rows";
  if (int rc = check_sizes(who, rows, cols, dtype)) return rc;
  FMOE_REQUIRE(activation == FMOE_ACT_NONE || activation == FMOE_ACT_GELU, "%s: bad activation %d",
               who, activation);
  FMOE_REQUIRE(rows == 0 || d_x, "%s: null device pointer", who);
  FMOE_REQUIRE(x_row_stride >= 0, "%s: negative row stride", who);
  if (int rc = check_rows8(who, d_q, q_stride, d_scales, rows, cols)) return rc;
  if (rows == 0) return FMOE_OK;
  const RowsArgs a{d_x, x_row_stride, rows, cols, static_cast<uint8_t*>(d_q), q_stride,
                   fmoe_host::round_up(cols, kRowsPitch), d_scales};
  hipStream_t s = static_cast<hipStream_t>(stream);
  by_float(dtype, [&](auto t) {
    using T = decltype(t);
    auto with = [&](auto act) {
      constexpr bool kG = decltype(act)::value;
      if (cols > kMaxRegCols) {
        hipLaunchKernelGGL((k_rows8_long<T, kG>), dim3((unsigned)rows), dim3(1024), 0, s, a);
        return;
      }
      by_cols(cols, [&](auto th, auto v) {
        constexpr int kT = decltype(th)::value;
        hipLaunchKernelGGL((k_rows8<T, kG, kT, decltype(v)::value>), row_grid<kT>(rows),
                           dim3(group_threads<kT>()), 0, s, a);
      });
    };
    if (activation == FMOE_ACT_GELU) with(std::true_type{});
    else with(std::false_type{});
  });
  return fmoe_host::check_launch(who);
}
