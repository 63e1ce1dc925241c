// The norms between two blocks: the one after a block, its gate and residual scale, the addition to the
// stream, and the one before the next block; forward and backward.
//
//   a = x * cx * post,  cx = 1 / sqrt(mean(x^2) + eps)          x: the block's output
//   h = residual + scale * gate * a, rounded to x's type: the stream as it is stored
//   y = h * ch * pre,   ch = 1 / sqrt(mean(h^2) + eps)          in fp32, rounded once
//
// gate: none, or [G, cols], a row for each of G equal runs of rows.  Backward, with x^ = x cx, h^ = h ch, t = gy pre
// and w = scale gate post:
//   grad_residual = R = gh + ch (t - h^ mean(t h^))
//   grad_x = cx (R w - x^ mean(R w x^))
//   grad_pre = sum over rows of gy h^
//   with A = sum over a run's rows of R x^:  grad_gate = scale post A,  grad_post = sum over runs of scale gate A
// so both hang on one sum a column.  Row sums need one round over the threads of a row, not two: the second
// mean is (sum(w (gh + ch t) x^) - ch mean(t h^) sum(w h^ x^)) / cols.
#include "rows8.h"

#include <algorithm>
#include <cmath>

namespace fmoe {

struct SandwichArgs {
  const void *x, *residual;
  int64_t x_stride, r_stride;  // elements
  const void *post, *pre, *gate;  // pre, gate: or null
  int w_dtype, gate_dtype;        // of post and pre; of the gate
  int64_t rows, cols, run;        // run: rows that share a row of the gate
  float scale, eps;
  void *h, *y;   // packed; y null without pre
  int stream_y;  // store y past the caches
  float* rstd;   // [rows, 2], or null
};

// Eight values of a parameter, which has the rows' type or fp32.
template <typename T> __device__ __forceinline__ void load_param(const void* p, int dtype, int64_t row_at, int64_t col,
                                                                 int64_t n, float* f) {
  if (dtype == FMOE_F32)
    Eight<float>::V::cvt(Eight<float>::template load<false>(static_cast<const float*>(p) + row_at, col, n), f);
  else if constexpr (!std::is_same<T, float>::value)
    Eight<T>::V::cvt(Eight<T>::template load<false>(static_cast<const T*>(p) + row_at, col, n), f);
}

template <int THREADS> constexpr int rows_of() { return THREADS < kGroup ? kGroup / THREADS : 1; }
template <int THREADS> constexpr int threads_of() { return THREADS < kGroup ? kGroup : THREADS; }

// The compiler would keep the converted values over the sums, which takes twice the registers; now it
// converts them again.
template <typename R> __device__ __forceinline__ void opaque(R& raw, int words) {
#pragma unroll
  for (int i = 0; i < words; ++i) {
    uint32_t w = raw[i];
    asm volatile("" : "+v"(w));
    raw[i] = w;
  }
}

// 64 registers, so that two workgroups of 1024 threads share a CU (4096 x 16384: 102 us, one with 74 registers 120).  The
// others are on a CU often enough as they are, and lose by the spills (4096 x 7168: 48 us, with 64 registers 56).
template <typename T, int THREADS, int VPT> constexpr bool two_on_a_cu() {
  return THREADS == 1024 && VPT == 2 && ElemInfo<T>::kBytes == 2;
}

// A row lies in the registers of THREADS threads, VPT vectors of eight columns each.
template <typename T, int THREADS, int VPT>
__global__ __launch_bounds__(threads_of<THREADS>(), (two_on_a_cu<T, THREADS, VPT>() ? 8 : 1)) void k_sandwich(SandwichArgs a) {
  __shared__ float lds[2][16];
  using V = Eight<T>;
  const int64_t row = (int64_t)blockIdx.x * rows_of<THREADS>() + threadIdx.x / THREADS;
  if (row >= a.rows) return;  // whole waves (THREADS == 64) or the whole workgroup
  const int tid = threadIdx.x % THREADS;
  const T* x = static_cast<const T*>(a.x) + row * a.x_stride;
  const T* r = static_cast<const T*>(a.residual) + row * a.r_stride;
  typename V::raw_t xr[VPT], rr[VPT];
#pragma unroll
  for (int v = 0; v < VPT; ++v) {
    xr[v] = V::template load<true>(x, (v * THREADS + tid) * 8, a.cols);
    rr[v] = V::template load<true>(r, (v * THREADS + tid) * 8, a.cols);
  }
  const int64_t gate_at = a.gate ? row / a.run * a.cols : 0;
  float w[VPT][8];
#pragma unroll
  for (int v = 0; v < VPT; ++v) {
    load_param<T>(a.post, a.w_dtype, 0, (v * THREADS + tid) * 8, a.cols, w[v]);
    float g[8];
    if (a.gate) load_param<T>(a.gate, a.gate_dtype, gate_at, (v * THREADS + tid) * 8, a.cols, g);
#pragma unroll
    for (int i = 0; i < 8; ++i) w[v][i] *= a.gate ? a.scale * g[i] : a.scale;
  }
  float sum = 0.f;
#pragma unroll
  for (int v = 0; v < VPT; ++v) {
    float f[8];
    V::V::cvt(xr[v], f);
#pragma unroll
    for (int i = 0; i < 8; ++i) sum = __builtin_fmaf(f[i], f[i], sum);
  }
  const float cx = 1.0f / sqrtf(group_sum<THREADS>(sum, lds[0]) / (float)a.cols + a.eps);
  sum = 0.f;
#pragma unroll
  for (int v = 0; v < VPT; ++v) {
    float f[8], s[8];
    opaque(xr[v], V::kWords);
    V::V::cvt(xr[v], f);
    V::V::cvt(rr[v], s);
#pragma unroll
    for (int i = 0; i < 8; ++i) s[i] = __builtin_fmaf(f[i] * cx, w[v][i], s[i]);
    xr[v] = V::V::pack(s);
    V::store(static_cast<T*>(a.h) + row * a.cols, (v * THREADS + tid) * 8, a.cols, xr[v]);
    V::V::cvt(xr[v], f);  // the stream is normalised as it is stored
#pragma unroll
    for (int i = 0; i < 8; ++i) sum = __builtin_fmaf(f[i], f[i], sum);
  }
  if (!a.pre && !a.rstd) return;
  float ch = 0.f;
  if (a.pre) {
#pragma unroll
    for (int v = 0; v < VPT; ++v) load_param<T>(a.pre, a.w_dtype, 0, (v * THREADS + tid) * 8, a.cols, w[v]);
    ch = 1.0f / sqrtf(group_sum<THREADS>(sum, lds[1]) / (float)a.cols + a.eps);
    T* y = static_cast<T*>(a.y) + row * a.cols;
#pragma unroll
    for (int v = 0; v < VPT; ++v) {
      float f[8];
      opaque(xr[v], V::kWords);
      V::V::cvt(xr[v], f);
#pragma unroll
      for (int i = 0; i < 8; ++i) f[i] = f[i] * ch * w[v][i];
      const typename V::raw_t q = V::V::pack(f);
      if (a.stream_y) V::template store<true>(y, (v * THREADS + tid) * 8, a.cols, q);
      else V::store(y, (v * THREADS + tid) * 8, a.cols, q);
    }
  }
  if (a.rstd && tid == 0) {
    a.rstd[2 * row] = cx;
    a.rstd[2 * row + 1] = ch;
  }
}

// Rows longer than the registers hold: the same steps, each over the row again.  A thread reads back only what it
// wrote or read itself.
template <typename T> __global__ __launch_bounds__(1024) void k_sandwich_long(SandwichArgs a) {
  __shared__ float lds[2][16];
  using V = Eight<T>;
  constexpr int kThreads = 1024;
  const int64_t row = blockIdx.x;
  const T* x = static_cast<const T*>(a.x) + row * a.x_stride;
  const T* r = static_cast<const T*>(a.residual) + row * a.r_stride;
  T* h = static_cast<T*>(a.h) + row * a.cols;
  const int64_t gate_at = a.gate ? row / a.run * a.cols : 0;
  float sum = 0.f;
  for (int64_t col = threadIdx.x * 8; col < a.cols; col += kThreads * 8) {
    float f[8];
    V::V::cvt(V::template load<false>(x, col, a.cols), f);
#pragma unroll
    for (int i = 0; i < 8; ++i) sum = __builtin_fmaf(f[i], f[i], sum);
  }
  const float cx = 1.0f / sqrtf(group_sum<kThreads>(sum, lds[0]) / (float)a.cols + a.eps);
  sum = 0.f;
  for (int64_t col = threadIdx.x * 8; col < a.cols; col += kThreads * 8) {
    float f[8], s[8], w[8], g[8];
    V::V::cvt(V::template load<false>(x, col, a.cols), f);
    V::V::cvt(V::template load<false>(r, col, a.cols), s);
    load_param<T>(a.post, a.w_dtype, 0, col, a.cols, w);
    if (a.gate) load_param<T>(a.gate, a.gate_dtype, gate_at, col, a.cols, g);
#pragma unroll
    for (int i = 0; i < 8; ++i)
      s[i] = __builtin_fmaf(f[i] * cx, w[i] * (a.gate ? a.scale * g[i] : a.scale), s[i]);
    const typename V::raw_t p = V::V::pack(s);
    V::store(h, col, a.cols, p);
    V::V::cvt(p, f);
#pragma unroll
    for (int i = 0; i < 8; ++i) sum = __builtin_fmaf(f[i], f[i], sum);
  }
  float ch = 0.f;
  if (a.pre) {
    ch = 1.0f / sqrtf(group_sum<kThreads>(sum, lds[1]) / (float)a.cols + a.eps);
    for (int64_t col = threadIdx.x * 8; col < a.cols; col += kThreads * 8) {
      float f[8], p[8];
      V::V::cvt(V::template load<false>(h, col, a.cols), f);
      load_param<T>(a.pre, a.w_dtype, 0, col, a.cols, p);
#pragma unroll
      for (int i = 0; i < 8; ++i) f[i] = f[i] * ch * p[i];
      V::store(static_cast<T*>(a.y) + row * a.cols, col, a.cols, V::V::pack(f));
    }
  }
  if (a.rstd && threadIdx.x == 0) {
    a.rstd[2 * row] = cx;
    a.rstd[2 * row + 1] = ch;
  }
}

struct SandwichBwdArgs {
  const void *gy, *gh;  // one of them may be null
  const void *x, *h;
  int64_t gy_stride, gh_stride, x_stride;  // elements; h is packed
  const void *post, *pre, *gate;
  int w_dtype, gate_dtype;
  const float* rstd;  // [rows, 2]
  int64_t rows, cols, run, runs;
  float scale;
  void *gx, *gr;    // packed; null where not wanted
  float* partials;  // [workgroups, 2, cols]: A (or the sum of scale gate A of whole runs), and grad_pre's part; or null
  void* ggate;      // [runs, cols], written here where a unit takes whole runs; else null
  int64_t units;    // rows in flight
  int64_t split;    // units that share a run, whole workgroups of them; 0: a unit takes whole runs, unit, unit + units, ...
  float* means;     // [rows]: mean(t h^), of rows that the registers do not hold
};

// Three sums over the threads of a row; `lds` holds them for every wave.
template <int THREADS> __device__ __forceinline__ void group_sum3(float* s, float (*lds)[16]) {
#pragma unroll
  for (int i = 0; i < 3; ++i) s[i] = wave_sum(s[i]);
  if constexpr (THREADS > kWave) {
    if ((threadIdx.x & (kWave - 1)) == 0)
#pragma unroll
      for (int i = 0; i < 3; ++i) lds[i][threadIdx.x / kWave] = s[i];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 3; ++i) {
      s[i] = lds[i][0];
#pragma unroll
      for (int w = 1; w < THREADS / kWave; ++w) s[i] += lds[i][w];
    }
  }
}

// The rows of a unit: of a run that `split` units share, every split-th; else all rows of its runs.
struct UnitRows {
  int64_t run, row, end, step;
  __device__ __forceinline__ UnitRows(const SandwichBwdArgs& a, int64_t unit) {
    run = a.split ? unit / a.split : unit;
    row = run * a.run + (a.split ? unit % a.split : 0);
    end = run < a.runs ? (run + 1) * a.run : 0;
    step = a.split ? a.split : 1;
  }
};

// A unit (the threads that hold a row) keeps its parts of the column sums, in registers or, for the longest rows
// (LDS_SUMS), in LDS, each thread its own: one pass over the four inputs, whatever the number of rows.  HBM bounds it: 12 bytes
// an element in 16 bits, 4096 x 16384 in 146 us: 5.5 TB/s.  In fp32, 2048 x 8192 takes 83 us: 4.9 TB/s; rows of 16384 do not fit
// the registers by 42 a thread, which pass through scratch memory: 2048 of them take 190 us, 4.3 TB/s.
// WHOLE: units take whole runs, write each one's gate's gradient and keep the sum of scale gate A in LDS.  Where a unit is a
// wave, the workgroup's four join their parts.
template <typename T, int THREADS, int VPT, bool WHOLE, bool LDS_SUMS>
__global__ __launch_bounds__(threads_of<THREADS>()) void k_sandwich_bwd(SandwichBwdArgs a) {
  static_assert(!(WHOLE && LDS_SUMS), "three sums do not fit");
  typedef float f32x4 __attribute__((ext_vector_type(4)));
  constexpr int kRows = rows_of<THREADS>(), kThreads = threads_of<THREADS>();
  constexpr int kA = WHOLE || LDS_SUMS || kRows > 1 ? VPT * 2 : 1, kB = LDS_SUMS || kRows > 1 ? VPT * 2 : 1;
  __shared__ float lds[2][3][16];
  __shared__ f32x4 sum_a[kA][kThreads], sum_b[kB][kThreads];
  using V = Eight<T>;
  const int64_t unit = (int64_t)blockIdx.x * kRows + threadIdx.x / THREADS;  // the grid has just the units
  const int tid = threadIdx.x % THREADS, me = threadIdx.x;
  float pre[VPT][8], w[VPT][8], A[LDS_SUMS ? 1 : VPT][8], B[LDS_SUMS ? 1 : VPT][8];
#pragma unroll
  for (int v = 0; v < VPT; ++v) {
    if (a.gy) load_param<T>(a.pre, a.w_dtype, 0, (v * THREADS + tid) * 8, a.cols, pre[v]);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if (!a.gy) pre[v][i] = 0.f;
      if constexpr (!LDS_SUMS) A[v][i] = B[v][i] = 0.f;
    }
    if constexpr (WHOLE || LDS_SUMS) sum_a[2 * v][me] = sum_a[2 * v + 1][me] = f32x4{0.f, 0.f, 0.f, 0.f};
    if constexpr (LDS_SUMS) sum_b[2 * v][me] = sum_b[2 * v + 1][me] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  // s += p * q, where a sum of this thread's lies in LDS
  auto add = [&](f32x4 (*s)[kThreads], int v, const float* p, const float* q) {
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      f32x4 t = s[2 * v + j][me];
#pragma unroll
      for (int i = 0; i < 4; ++i) t[i] = __builtin_fmaf(p[4 * j + i], q[4 * j + i], t[i]);
      s[2 * v + j][me] = t;
    }
  };
  const float inv_cols = 1.0f / (float)a.cols;
  int turn = 0;
  for (UnitRows u(a, unit); u.run < a.runs;) {
#pragma unroll
    for (int v = 0; v < VPT; ++v) {
      load_param<T>(a.post, a.w_dtype, 0, (v * THREADS + tid) * 8, a.cols, w[v]);
      float g[8];
      if (a.gate) load_param<T>(a.gate, a.gate_dtype, u.run * a.cols, (v * THREADS + tid) * 8, a.cols, g);
#pragma unroll
      for (int i = 0; i < 8; ++i) w[v][i] *= a.gate ? a.scale * g[i] : a.scale;
    }
    for (; u.row < u.end; u.row += u.step, turn ^= 1) {
      typename V::raw_t gyr[VPT], ghr[VPT], xr[VPT], hr[VPT];
#pragma unroll
      for (int v = 0; v < VPT; ++v) {
        const int64_t col = (v * THREADS + tid) * 8;
        gyr[v] = a.gy ? V::template load<true>(static_cast<const T*>(a.gy) + u.row * a.gy_stride, col, a.cols) : V::zero();
        hr[v] = V::template load<true>(static_cast<const T*>(a.h) + u.row * a.cols, col, a.cols);
        ghr[v] = a.gh ? V::template load<true>(static_cast<const T*>(a.gh) + u.row * a.gh_stride, col, a.cols) : V::zero();
        xr[v] = V::template load<true>(static_cast<const T*>(a.x) + u.row * a.x_stride, col, a.cols);
      }
      const float cx = a.rstd[2 * u.row], ch = a.rstd[2 * u.row + 1];
      float s[3] = {0.f, 0.f, 0.f};
#pragma unroll
      for (int v = 0; v < VPT; ++v) {
        float gy[8], gh[8], x[8], h[8];
        V::V::cvt(gyr[v], gy);
        V::V::cvt(ghr[v], gh);
        V::V::cvt(xr[v], x);
        V::V::cvt(hr[v], h);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          h[i] *= ch;
          const float t = gy[i] * pre[v][i], wx = w[v][i] * (x[i] * cx);
          if constexpr (!LDS_SUMS) B[v][i] = __builtin_fmaf(gy[i], h[i], B[v][i]);
          s[0] = __builtin_fmaf(t, h[i], s[0]);
          s[1] = __builtin_fmaf(wx, __builtin_fmaf(ch, t, gh[i]), s[1]);
          s[2] = __builtin_fmaf(wx, h[i], s[2]);
        }
        if constexpr (LDS_SUMS) add(sum_b, v, gy, h);
      }
      // the waves' words of LDS, used in turn: a thread that is a row ahead writes the other
      group_sum3<THREADS>(s, lds[turn]);
      const float m = s[0] * inv_cols;
      const float mx = __builtin_fmaf(-ch * m, s[2], s[1]) * inv_cols;
#pragma unroll
      for (int v = 0; v < VPT; ++v) {
        opaque(gyr[v], V::kWords);
        opaque(ghr[v], V::kWords);
        opaque(xr[v], V::kWords);
        opaque(hr[v], V::kWords);
      }
#pragma unroll
      for (int v = 0; v < VPT; ++v) {
        float gy[8], r[8], x[8], h[8];
        V::V::cvt(gyr[v], gy);
        V::V::cvt(ghr[v], r);
        V::V::cvt(xr[v], x);
        V::V::cvt(hr[v], h);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          x[i] *= cx;
          r[i] = __builtin_fmaf(ch, __builtin_fmaf(-(h[i] * ch), m, gy[i] * pre[v][i]), r[i]);
          if constexpr (!LDS_SUMS) A[v][i] = __builtin_fmaf(r[i], x[i], A[v][i]);
        }
        if constexpr (LDS_SUMS) add(sum_a, v, r, x);
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = cx * __builtin_fmaf(-x[i], mx, r[i] * w[v][i]);
        const int64_t col = (v * THREADS + tid) * 8;
        if (a.gr) V::template store<true>(static_cast<T*>(a.gr) + u.row * a.cols, col, a.cols, V::V::pack(r));
        if (a.gx) V::template store<true>(static_cast<T*>(a.gx) + u.row * a.cols, col, a.cols, V::V::pack(x));
      }
    }
    if constexpr (!WHOLE) {
      break;
    } else {
#pragma unroll
      for (int v = 0; v < VPT; ++v) {
        const int64_t col = (v * THREADS + tid) * 8;
        float g[8], post[8];
        load_param<T>(a.gate, a.gate_dtype, u.run * a.cols, col, a.cols, g);
#pragma unroll
        for (int i = 0; i < 8; ++i) g[i] *= a.scale;
        add(sum_a, v, g, A[v]);
        load_param<T>(a.post, a.w_dtype, 0, col, a.cols, post);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          g[i] = a.scale * post[i] * A[v][i];
          A[v][i] = 0.f;
        }
        if (!a.ggate) continue;
        if (a.gate_dtype == FMOE_F32)
          Eight<float>::store(static_cast<float*>(a.ggate) + u.run * a.cols, col, a.cols, Eight<float>::V::pack(g));
        else V::store(static_cast<T*>(a.ggate) + u.run * a.cols, col, a.cols, V::V::pack(g));
      }
      u.run += a.units;
      u.row = u.run * a.run;
      u.end = u.row + a.run;
    }
  }
  if (!a.partials) return;
  // the four units of a workgroup have rows of one run (or whole runs each, whose sums are weighted by now)
  if constexpr (kRows > 1) {
#pragma unroll
    for (int v = 0; v < VPT; ++v)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        if constexpr (!WHOLE) sum_a[2 * v + j][me] = f32x4{A[v][4 * j], A[v][4 * j + 1], A[v][4 * j + 2], A[v][4 * j + 3]};
        sum_b[2 * v + j][me] = f32x4{B[v][4 * j], B[v][4 * j + 1], B[v][4 * j + 2], B[v][4 * j + 3]};
      }
    __syncthreads();
    if (threadIdx.x >= THREADS) return;
  }
  float* out = a.partials + (int64_t)blockIdx.x * 2 * a.cols;
#pragma unroll
  for (int v = 0; v < VPT; ++v) {
    float p[8], q[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      p[i] = kA > 1 ? sum_a[kA > 1 ? 2 * v + i / 4 : 0][me][i % 4] : A[LDS_SUMS ? 0 : v][i];
      q[i] = kB > 1 ? sum_b[kB > 1 ? 2 * v + i / 4 : 0][me][i % 4] : B[LDS_SUMS ? 0 : v][i];
      if constexpr (kRows > 1) {
#pragma unroll
        for (int r = 1; r < kRows; ++r) {
          p[i] += sum_a[kA > 1 ? 2 * v + i / 4 : 0][r * THREADS + me][i % 4];
          q[i] += sum_b[kB > 1 ? 2 * v + i / 4 : 0][r * THREADS + me][i % 4];
        }
      }
    }
    const int64_t col = (v * THREADS + tid) * 8;
    Eight<float>::store(out, col, a.cols, Eight<float>::V::pack(p));
    Eight<float>::store(out + a.cols, col, a.cols, Eight<float>::V::pack(q));
  }
}

// Rows longer than the registers hold: the gradients of x and the residual row by row, then the column sums.
template <typename T> __global__ __launch_bounds__(1024) void k_sandwich_bwd_long(SandwichBwdArgs a) {
  __shared__ float lds[3][16];
  using V = Eight<T>;
  constexpr int kThreads = 1024;
  const int64_t row = blockIdx.x, gate_at = a.gate ? row / a.run * a.cols : 0;
  const float cx = a.rstd[2 * row], ch = a.rstd[2 * row + 1];
  float gy[8], gh[8], x[8], h[8], pre[8], w[8];
  auto read = [&](int64_t col) {
    V::V::cvt(a.gy ? V::template load<false>(static_cast<const T*>(a.gy) + row * a.gy_stride, col, a.cols) : V::zero(), gy);
    V::V::cvt(a.gh ? V::template load<false>(static_cast<const T*>(a.gh) + row * a.gh_stride, col, a.cols) : V::zero(), gh);
    V::V::cvt(V::template load<false>(static_cast<const T*>(a.x) + row * a.x_stride, col, a.cols), x);
    V::V::cvt(V::template load<false>(static_cast<const T*>(a.h) + row * a.cols, col, a.cols), h);
    load_param<T>(a.post, a.w_dtype, 0, col, a.cols, w);
    float g[8];
    if (a.gate) load_param<T>(a.gate, a.gate_dtype, gate_at, col, a.cols, g);
    if (a.gy) load_param<T>(a.pre, a.w_dtype, 0, col, a.cols, pre);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      w[i] *= a.gate ? a.scale * g[i] : a.scale;
      if (!a.gy) pre[i] = 0.f;
    }
  };
  float s[3] = {0.f, 0.f, 0.f};
  for (int64_t col = threadIdx.x * 8; col < a.cols; col += kThreads * 8) {
    read(col);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float t = gy[i] * pre[i], hh = h[i] * ch, wx = w[i] * (x[i] * cx);
      s[0] = __builtin_fmaf(t, hh, s[0]);
      s[1] = __builtin_fmaf(wx, __builtin_fmaf(ch, t, gh[i]), s[1]);
      s[2] = __builtin_fmaf(wx, hh, s[2]);
    }
  }
  group_sum3<kThreads>(s, lds);
  const float inv_cols = 1.0f / (float)a.cols, m = s[0] * inv_cols;
  const float mx = __builtin_fmaf(-ch * m, s[2], s[1]) * inv_cols;
  if (threadIdx.x == 0) a.means[row] = m;
  for (int64_t col = threadIdx.x * 8; col < a.cols; col += kThreads * 8) {
    read(col);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      gh[i] = __builtin_fmaf(ch, __builtin_fmaf(-(h[i] * ch), m, gy[i] * pre[i]), gh[i]);
      x[i] = cx * __builtin_fmaf(-(x[i] * cx), mx, gh[i] * w[i]);
    }
    if (a.gr) V::store(static_cast<T*>(a.gr) + row * a.cols, col, a.cols, V::V::pack(gh));
    if (a.gx) V::store(static_cast<T*>(a.gx) + row * a.cols, col, a.cols, V::V::pack(x));
  }
}

template <typename T> __global__ __launch_bounds__(kGroup) void k_sandwich_bwd_long_w(SandwichBwdArgs a) {
  using V = Eight<T>;
  const int64_t unit = blockIdx.x;
  const int64_t col = ((int64_t)blockIdx.y * kGroup + threadIdx.x) * 8;
  if (col >= a.cols) return;
  float pre[8], post[8], A[8], B[8], P[8];
  load_param<T>(a.post, a.w_dtype, 0, col, a.cols, post);
  if (a.gy) load_param<T>(a.pre, a.w_dtype, 0, col, a.cols, pre);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    A[i] = B[i] = P[i] = 0.f;
    if (!a.gy) pre[i] = 0.f;
  }
  for (UnitRows u(a, unit); u.run < a.runs;) {
    for (; u.row < u.end; u.row += u.step) {
      float gy[8], r[8], x[8], h[8];
      V::V::cvt(a.gy ? V::template load<false>(static_cast<const T*>(a.gy) + u.row * a.gy_stride, col, a.cols) : V::zero(), gy);
      V::V::cvt(a.gh ? V::template load<false>(static_cast<const T*>(a.gh) + u.row * a.gh_stride, col, a.cols) : V::zero(), r);
      V::V::cvt(V::template load<false>(static_cast<const T*>(a.x) + u.row * a.x_stride, col, a.cols), x);
      V::V::cvt(V::template load<false>(static_cast<const T*>(a.h) + u.row * a.cols, col, a.cols), h);
      const float cx = a.rstd[2 * u.row], ch = a.rstd[2 * u.row + 1], m = a.means[u.row];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float hh = h[i] * ch;
        r[i] = __builtin_fmaf(ch, __builtin_fmaf(-hh, m, gy[i] * pre[i]), r[i]);
        A[i] = __builtin_fmaf(r[i], x[i] * cx, A[i]);
        B[i] = __builtin_fmaf(gy[i], hh, B[i]);
      }
    }
    if (a.split) break;
    float g[8];
    load_param<T>(a.gate, a.gate_dtype, u.run * a.cols, col, a.cols, g);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      P[i] = __builtin_fmaf(a.scale * g[i], A[i], P[i]);
      g[i] = a.scale * post[i] * A[i];
      A[i] = 0.f;
    }
    if (a.ggate) {
      if (a.gate_dtype == FMOE_F32)
        Eight<float>::store(static_cast<float*>(a.ggate) + u.run * a.cols, col, a.cols, Eight<float>::V::pack(g));
      else V::store(static_cast<T*>(a.ggate) + u.run * a.cols, col, a.cols, V::V::pack(g));
    }
    u.run += a.units;
    u.row = u.run * a.run;
    u.end = u.row + a.run;
  }
  float* out = a.partials + unit * 2 * a.cols;
  Eight<float>::store(out, col, a.cols, Eight<float>::V::pack(a.split ? A : P));
  Eight<float>::store(out + a.cols, col, a.cols, Eight<float>::V::pack(B));
}

struct JoinArgs {
  const float* partials;  // [parts, 2, cols]
  int64_t parts, split, runs, cols;  // split: parts of a run; 0: the parts are of whole runs
  const void *post, *gate;
  void *gpost, *gpre, *ggate;  // null where not wanted (ggate: where units took whole runs)
  int w_dtype, gate_dtype;
  float scale;
};
__device__ __forceinline__ void store_param(void* p, int dtype, int64_t i, float v) {
  if (dtype == FMOE_F32) static_cast<float*>(p)[i] = v;
  else if (dtype == FMOE_BF16) st1(static_cast<bf16_t*>(p) + i, v);
  else st1(static_cast<f16_t*>(p) + i, v);
}

// Each column's sums in one fixed order: a workgroup takes 32 columns, 128 bytes of a part, each of its 32 slots every
// so many of the parts, eight at a time on their way; several runs share the slots out.  512 parts of 4096 columns take 6.7 us
// (with 64 columns 7.5, with 16 8.5), 256 of 16384 9.0 (8.7, 16.7); one after the other they took 20.
constexpr int kJoinThreads = 1024, kJoinCols = 32, kSlots = kJoinThreads / kJoinCols, kBatch = 8;
__global__ __launch_bounds__(kJoinThreads) void k_sandwich_join(JoinArgs a) {
  __shared__ float lds[2][kSlots][kJoinCols];
  const int c = threadIdx.x % kJoinCols, slot = threadIdx.x / kJoinCols;
  const int64_t col = (int64_t)blockIdx.x * kJoinCols + c;
  const bool here = col < a.cols;
  const float post = here ? load_weight(a.post, a.w_dtype, col) : 0.f;
  const int64_t runs = a.split ? a.runs : 1, per = a.split ? a.split : a.parts;
  int share = kSlots;  // slots of a run
  while (share > 1 && share * runs > kSlots) share /= 2;
  const int sub = slot % share;
  // v of the slots slot, slot + 1, ... slot + n - 1, where slot is a multiple of n; the whole workgroup calls it
  auto together = [&](int n, int which, float v) {
    lds[which][slot][c] = v;
    __syncthreads();
    for (n /= 2; n >= 1; n /= 2) {
      if ((slot & (2 * n - 1)) < n) lds[which][slot][c] = v += lds[which][slot + n][c];
      __syncthreads();
    }
    return v;
  };
  float s = 0.f, b = 0.f;
  for (int64_t r0 = 0; r0 < runs; r0 += kSlots / share) {
    const int64_t run = r0 + slot / share;
    float A = 0.f;
    if (here && run < runs) {
      const int64_t end = (run + 1) * per;
      for (int64_t u = run * per + sub; u < end; u += kBatch * share) {
        float va[kBatch], vb[kBatch];
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {
          const float* at = a.partials + min(u + i * share, end - 1) * 2 * a.cols + col;
          va[i] = at[0];
          vb[i] = at[a.cols];
        }
#pragma unroll
        for (int i = 0; i < kBatch; ++i)
          if (u + i * share < end) {
            A += va[i];
            b += vb[i];
          }
      }
    }
    if (share > 1) A = together(share, 0, A);
    if (here && run < runs && sub == 0) {
      if (!a.split) s = A;  // of whole runs: weighted already
      else {
        if (a.ggate) store_param(a.ggate, a.gate_dtype, run * a.cols + col, a.scale * post * A);
        s = __builtin_fmaf(a.gate ? a.scale * load_weight(a.gate, a.gate_dtype, run * a.cols + col) : a.scale, A, s);
      }
    }
  }
  s = together(kSlots, 0, s);
  b = together(kSlots, 1, b);
  if (slot != 0 || !here) return;
  if (a.gpost) store_param(a.gpost, a.w_dtype, col, s);
  if (a.gpre) store_param(a.gpre, a.w_dtype, col, b);
}

}  // namespace fmoe

using namespace fmoe;

namespace {

constexpr int64_t kMaxRegCols = 16384;          // columns that the largest register variant holds
constexpr int64_t kMaxCols = int64_t(1) << 26;  // 2048 columns for each of a grid's 2^15 in y
constexpr int64_t kMaxSumCols = 8192;           // columns whose sums of whole runs fit

template <typename F> void by_type(int dtype, F&& f) {
  if (dtype == FMOE_F32) f(float{});
  else if (dtype == FMOE_BF16) f(bf16_t{});
  else f(f16_t{});
}
template <int N> using Int = std::integral_constant<int, N>;

// Calls f(threads, vectors) with the variant that holds a row.  Few rows are given more threads: then a row's
// latency counts (8 x 7168: 4.8 us with 1024 threads, 5.2 with 512, 6.3 with 256; 4096 x 7168: 52, 48 and 51).
constexpr int64_t kFewRows = 512;
template <typename F> void by_cols(int64_t rows, int64_t cols, F&& f) {
  const int64_t v = (cols + 7) / 8;
  if (v <= 64) f(Int<64>{}, Int<1>{});
  else if (v <= 128) f(Int<64>{}, Int<2>{});
  else if (v <= 256) f(Int<64>{}, Int<4>{});
  else if (v <= 512) f(Int<256>{}, Int<2>{});
  else if (v <= 1024 && rows <= kFewRows) f(Int<1024>{}, Int<1>{});
  else if (v <= 1024) f(Int<512>{}, Int<2>{});
  else f(Int<1024>{}, Int<2>{});
}
template <typename F> void by_cols_backward(int64_t cols, F&& f) {
  const int64_t v = (cols + 7) / 8;
  if (v <= 64) f(Int<64>{}, Int<1>{});
  else if (v <= 128) f(Int<64>{}, Int<2>{});
  else if (v <= 256) f(Int<256>{}, Int<1>{});
  else if (v <= 512) f(Int<256>{}, Int<2>{});
  else if (v <= 1024) f(Int<512>{}, Int<2>{});
  else f(Int<1024>{}, Int<2>{});
}

int check_sandwich(const char* who, int64_t rows, int64_t cols, int dtype, int w_dtype, const void* gate,
                   int gate_dtype, int64_t gate_rows, const void* post) {
  FMOE_REQUIRE(rows >= 0 && cols >= 1, "%s: bad sizes rows=%lld columns=%lld", who, (long long)rows, (long long)cols);
  FMOE_REQUIRE(fmoe_host::is_float_dtype(dtype), "%s: bad dtype %d", who, dtype);
  FMOE_REQUIRE(post, "%s: null device pointer", who);
  FMOE_REQUIRE(w_dtype == dtype || w_dtype == FMOE_F32, "%s: the weights must have the rows' dtype or fp32", who);
  FMOE_REQUIRE(!gate || gate_dtype == dtype || gate_dtype == FMOE_F32, "%s: the gate must have the rows' dtype or fp32",
               who);
  FMOE_REQUIRE(gate ? gate_rows >= 1 && rows % gate_rows == 0 : gate_rows == 0,
               "%s: %lld rows of the gate for %lld rows", who, (long long)gate_rows, (long long)rows);
  const int64_t threads = cols <= 2048 ? 64 : cols <= 8192 ? 512 : 1024;
  if (cols > kMaxCols || rows > ((int64_t(1) << 32) - 1024) / threads) {
    fmoe_host::set_error("%s: rows=%lld or columns=%lld too large", who, (long long)rows, (long long)cols);
    return FMOE_ERANGE;
  }
  return FMOE_OK;
}

template <int THREADS> dim3 grid_of(int64_t units) {
  constexpr int per = rows_of<THREADS>();
  return dim3((unsigned)((units + per - 1) / per));
}

// How the backward's rows are shared out.
struct Shares {
  int64_t groups;  // workgroups, as many parts of the column sums
  int64_t split;   // of them, those that share a run; 0: units take whole runs
  int64_t rows;    // rows in flight in a workgroup
  bool long_rows;  // the rows, then the columns
};
Shares shares_of(int64_t rows, int64_t cols, int64_t runs) {
  Shares s{0, 0, 1, cols > kMaxRegCols};
  if (rows == 0) return s;
  // Each workgroup's part is 8 bytes a column to write and to read again; two workgroups are on a CU together where rows are
  // short (with the join, bf16, 16384 x 2048: 83 us with 512 workgroups, 118 with 256, 91 with 1024; 16384 x 4096: 147, 194
  // and 156; 8192 x 7168: 155, 150 and 169; 4096 x 16384: 177, 164 and 198).
  const int64_t most = cols <= 4096 ? 512 : 256;
  const bool whole = runs >= most;
  s.long_rows |= whole && cols > kMaxSumCols;
  if (!s.long_rows && cols <= 1024) s.rows = 4;
  if (whole) {
    s.groups = std::min(most, (runs + s.rows - 1) / s.rows);
  } else {
    s.split = std::min(most / runs, (rows / runs + s.rows - 1) / s.rows);
    s.groups = s.split * runs;
  }
  return s;
}

}  // namespace

extern "C" int fmoe_sandwich_norm(const void* d_x, int64_t x_row_stride, const void* d_residual,
                                  int64_t residual_row_stride, const void* d_post, const void* d_pre,
                                  int weight_dtype, const void* d_gate, int gate_dtype, int64_t gate_rows,
                                  int64_t rows, int64_t cols, int dtype, float scale, float eps, void* d_h,
                                  void* d_y, float* d_rstd, void* stream) {
  fmoe_host::clear_error();
  const char* who = "fmoe_sandwich_norm";
  if (int rc = check_sandwich(who, rows, cols, dtype, weight_dtype, d_gate, gate_dtype, gate_rows, d_post)) return rc;
  FMOE_REQUIRE(x_row_stride >= 0 && residual_row_stride >= 0, "%s: negative row stride", who);
  FMOE_REQUIRE(std::isfinite(scale) && eps >= 0.f && std::isfinite(eps),
               "%s: the scale must be finite, eps finite and not negative", who);
  if (rows == 0) return FMOE_OK;
  FMOE_REQUIRE(d_x && d_residual && d_h && !d_pre == !d_y, "%s: null device pointer", who);
  const SandwichArgs a{d_x, d_residual, x_row_stride, residual_row_stride, d_post, d_pre, d_gate, weight_dtype,
                       gate_dtype, rows, cols, d_gate ? rows / gate_rows : rows, scale, eps, d_h, d_y,
                       rows * cols * fmoe_host::dtype_bytes(dtype) >= FMOE_STREAM_OUT_BYTES, d_rstd};
  hipStream_t s = static_cast<hipStream_t>(stream);
  by_type(dtype, [&](auto t) {
    using T = decltype(t);
    if (cols > kMaxRegCols) {
      hipLaunchKernelGGL((k_sandwich_long<T>), dim3((unsigned)rows), dim3(1024), 0, s, a);
      return;
    }
    by_cols(rows, cols, [&](auto th, auto v) {
      constexpr int kT = decltype(th)::value;
      hipLaunchKernelGGL((k_sandwich<T, kT, decltype(v)::value>), grid_of<kT>(rows), dim3(threads_of<kT>()), 0, s, a);
    });
  });
  return fmoe_host::check_launch(who);
}

extern "C" int64_t fmoe_sandwich_norm_backward_workspace_bytes(int64_t rows, int64_t cols, int64_t gate_rows) {
  if (rows < 0 || cols < 1 || gate_rows < 0 || (gate_rows && rows % gate_rows)) return -1;
  const Shares s = shares_of(rows, cols, std::max<int64_t>(gate_rows, 1));
  return std::max<int64_t>(s.groups, 1) * cols * 8 + (s.long_rows ? rows * 4 : 0);
}

extern "C" int fmoe_sandwich_norm_backward(const void* d_grad_y, int64_t gy_row_stride, const void* d_grad_h,
                                           int64_t gh_row_stride, const void* d_x, int64_t x_row_stride,
                                           const void* d_h, const void* d_post, const void* d_pre, int weight_dtype,
                                           const void* d_gate, int gate_dtype, int64_t gate_rows,
                                           const float* d_rstd, int64_t rows, int64_t cols, int dtype, float scale,
                                           void* d_grad_x, void* d_grad_residual, void* d_grad_post,
                                           void* d_grad_pre, void* d_grad_gate, void* d_workspace,
                                           int64_t workspace_bytes, void* stream) {
  fmoe_host::clear_error();
  const char* who = "fmoe_sandwich_norm_backward";
  if (int rc = check_sandwich(who, rows, cols, dtype, weight_dtype, d_gate, gate_dtype, gate_rows, d_post)) return rc;
  FMOE_REQUIRE(gy_row_stride >= 0 && gh_row_stride >= 0 && x_row_stride >= 0, "%s: negative row stride", who);
  FMOE_REQUIRE(rows == 0 || (d_x && d_h && d_rstd && (d_grad_y || d_grad_h)), "%s: null device pointer", who);
  FMOE_REQUIRE(!d_grad_y || d_pre, "%s: y's gradient needs its weight", who);
  FMOE_REQUIRE(!d_grad_gate || (d_gate && rows > 0), "%s: no gate or no rows to have its gradient from", who);
  const bool sums = d_grad_post || d_grad_pre || d_grad_gate;
  const int64_t need = fmoe_sandwich_norm_backward_workspace_bytes(rows, cols, gate_rows);
  const int64_t runs = d_gate ? gate_rows : 1;
  const Shares sh = shares_of(rows, cols, runs);
  FMOE_REQUIRE((!sums && !sh.long_rows) || (d_workspace && workspace_bytes >= need &&
                                            reinterpret_cast<uintptr_t>(d_workspace) % 16 == 0),
               "%s: needs an aligned workspace of %lld bytes", who, (long long)need);
  SandwichBwdArgs a{d_grad_y, d_grad_h, d_x, d_h, gy_row_stride, gh_row_stride, x_row_stride, d_post, d_pre, d_gate,
                    weight_dtype, gate_dtype, d_rstd, rows, cols, rows / runs, runs, scale, d_grad_x,
                    d_grad_residual, sums ? static_cast<float*>(d_workspace) : nullptr, nullptr, 0, 0, nullptr};
  a.units = sh.groups * sh.rows;
  a.split = sh.split * sh.rows;
  const bool whole = rows > 0 && !sh.split;
  if (whole) a.ggate = d_grad_gate;
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (rows > 0)
    by_type(dtype, [&](auto t) {
      using T = decltype(t);
      if (sh.long_rows) {
        a.means = static_cast<float*>(d_workspace) + sh.groups * 2 * cols;
        hipLaunchKernelGGL((k_sandwich_bwd_long<T>), dim3((unsigned)rows), dim3(1024), 0, s, a);
        if (sums)
          hipLaunchKernelGGL((k_sandwich_bwd_long_w<T>),
                             dim3((unsigned)a.units, (unsigned)((cols + kGroup * 8 - 1) / (kGroup * 8))), dim3(kGroup),
                             0, s, a);
        return;
      }
      by_cols_backward(cols, [&](auto th, auto v) {
        constexpr int kT = decltype(th)::value, kV = decltype(v)::value;
        constexpr bool kLds = kT == 1024;
        const dim3 grid((unsigned)sh.groups), block(threads_of<kT>());
        if constexpr (!kLds)
          if (whole) {
            hipLaunchKernelGGL((k_sandwich_bwd<T, kT, kV, true, false>), grid, block, 0, s, a);
            return;
          }
        hipLaunchKernelGGL((k_sandwich_bwd<T, kT, kV, false, kLds>), grid, block, 0, s, a);
      });
    });
  if (sums) {
    // without rows: no parts, and zeros
    const JoinArgs j{a.partials, sh.groups, sh.split, runs, cols, d_post, d_gate,
                     d_grad_post, d_grad_pre, whole ? nullptr : d_grad_gate, weight_dtype, gate_dtype, scale};
    hipLaunchKernelGGL(k_sandwich_join, dim3((unsigned)((cols + kJoinCols - 1) / kJoinCols)), dim3(kJoinThreads), 0, s, j);
  }
  return fmoe_host::check_launch(who);
}
