// Activations held in 8 bits from a training step's forward to its backward.
//
// Every block of 128 columns of a row has a scale of its own (rows8.h): 1.03 bytes an element
// instead of 2 or 4, each value within 1/254 of its block's largest.
//   compress        q, s of x; with GELU also a = gelu(x) of the exact x, or a alone
//   restore         q * s
//   GELU's backward held = q * s;  again = gelu(held);  grad = grad_a * gelu'(held)
//
// Bound by HBM: 16 lanes hold a block, eight columns each, so a block's maximum is four DPP
// rotations and every array is read or written once, 16 (bytes: 8) bytes a lane.
#include "rows8.h"

#include <algorithm>

namespace fmoe {

// Rows of a thread, which asks for all of them first: 32768 x 2048 in bf16 take 59.3 us (GELU and 8 bits), 34.5
// (8 bits) and 32.1 (back, through the caches), with one row 62.2, 36.8 and 35.1, with four 60.4, 34.3 and
// 31.8; GELU's backward gains nothing there, and 4 % at 4096 x 14336.  In fp32 restoring two takes 78 us,
// one 60.
template <typename T> constexpr int hold_rows() { return ElemInfo<T>::kBytes == 2 ? 2 : 1; }

// A workgroup is `1 << tx` vectors of eight columns wide and step = kGroup >> tx rows high, and goes
// on to the next `step` rows `each` times; `chunks` workgroups side by side cover a row.
struct HoldGrid {
  int tx, chunks, step, each;
  __device__ __forceinline__ bool place(int64_t rows, int64_t* row, int64_t* col) const {
    *row = (int64_t)(blockIdx.x / (unsigned)chunks) * step * each + (threadIdx.x >> tx);
    *col = ((int64_t)(blockIdx.x % (unsigned)chunks) * (1 << tx) + (threadIdx.x & ((1 << tx) - 1))) * 8;
    return *row < rows;
  }
};

struct HoldArgs {
  const void* x;      // compress: the rows; backward: grad_a
  int64_t x_stride;   // elements
  int64_t rows, cols, blocks;
  uint8_t* q;         // rows of q_stride bytes; null (compress) where only a is wanted
  int64_t q_stride;
  float* scales;      // packed [rows, blocks]
  void* out;          // compress: a; restore: x; backward: grad.  Packed.
  void* again;        // backward: gelu of the held rows, packed, or null
  int past;           // restore, backward: outputs go past the caches
  HoldGrid grid;
};

template <typename T>
__device__ __forceinline__ void put(const HoldArgs& a, void* to, int64_t row, int64_t col,
                                    typename Eight<T>::raw_t v) {
  T* p = static_cast<T*>(to) + row * a.cols;
  if (a.past) Eight<T>::template store<true>(p, col, a.cols, v);
  else Eight<T>::store(p, col, a.cols, v);
}

template <typename T, bool HOLD, bool GELU> __global__ __launch_bounds__(kGroup) void k_compress(HoldArgs a) {
  constexpr int ROWS = hold_rows<T>();
  int64_t row, col;
  using V = Eight<T>;
  // the lanes of a block stay together: a row's vectors beyond its last block are whole DPP rows
  if (!a.grid.place(a.rows, &row, &col) || col >= a.blocks * kHoldBlock) return;
  typename V::raw_t raw[ROWS];
#pragma unroll
  for (int r = 0; r < ROWS; ++r)
    raw[r] = V::template load<true>(
        static_cast<const T*>(a.x) + min(row + r * a.grid.step, a.rows - 1) * a.x_stride, col, a.cols);
#pragma unroll
  for (int r = 0; r < ROWS; ++r, row += a.grid.step) {
    if (row >= a.rows) return;
    float f[8];
    V::V::cvt(raw[r], f);
    if constexpr (HOLD) {
      float top = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) top = larger(top, f[i]);
      const Scale8 s = scale8(row_max(abs_bits(top)));
      if (col % kHoldBlock == 0) a.scales[row * a.blocks + col / kHoldBlock] = s.scale;
      *reinterpret_cast<u32x2*>(a.q + row * a.q_stride + col) = pack8(f, s);
    }
    if constexpr (GELU) {
#pragma unroll
      for (int i = 0; i < 8; ++i) f[i] = gelu<T>(f[i]);
      V::store(static_cast<T*>(a.out) + row * a.cols, col, a.cols, V::V::pack(f));
    }
  }
}

template <typename T> __global__ __launch_bounds__(kGroup) void k_restore(HoldArgs a) {
  constexpr int ROWS = hold_rows<T>();
  int64_t row, col;
  using V = Eight<T>;
  if (!a.grid.place(a.rows, &row, &col) || col >= a.cols) return;
  u32x2 q[ROWS];
  float scale[ROWS];
#pragma unroll
  for (int r = 0; r < ROWS; ++r) {
    const int64_t at = min(row + r * a.grid.step, a.rows - 1);
    q[r] = *reinterpret_cast<const u32x2*>(a.q + at * a.q_stride + col);
    scale[r] = a.scales[at * a.blocks + (a.blocks > 1 ? col / kHoldBlock : 0)];
  }
#pragma unroll
  for (int r = 0; r < ROWS; ++r, row += a.grid.step) {
    if (row >= a.rows) return;
    float f[8];
    unpack8(q[r], scale[r], f);
    put<T>(a, a.out, row, col, V::V::pack(f));
  }
}

template <typename T> __global__ __launch_bounds__(kGroup) void k_gelu_backward(HoldArgs a) {
  constexpr int ROWS = hold_rows<T>();
  int64_t row, col;
  using V = Eight<T>;
  if (!a.grid.place(a.rows, &row, &col) || col >= a.cols) return;
  u32x2 q[ROWS];
  float scale[ROWS];
  typename V::raw_t raw[ROWS];
#pragma unroll
  for (int r = 0; r < ROWS; ++r) {
    const int64_t at = min(row + r * a.grid.step, a.rows - 1);
    q[r] = *reinterpret_cast<const u32x2*>(a.q + at * a.q_stride + col);
    raw[r] = V::template load<true>(static_cast<const T*>(a.x) + at * a.x_stride, col, a.cols);
    scale[r] = a.scales[at * a.blocks + col / kHoldBlock];
  }
#pragma unroll
  for (int r = 0; r < ROWS; ++r, row += a.grid.step) {
    if (row >= a.rows) return;
    float f[8], g[8];
    unpack8(q[r], scale[r], f);
    V::V::cvt(raw[r], g);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float cdf = normal_cdf<T>(f[i]);
      g[i] *= gelu_slope(f[i], cdf);
      f[i] *= cdf;
    }
    if (a.again) put<T>(a, a.again, row, col, V::V::pack(f));
    put<T>(a, a.out, row, col, V::V::pack(g));
  }
}

}  // namespace fmoe

using namespace fmoe;

namespace {

// Fills in the grid and checks what every call has; *groups = 0 where there is nothing to do.  `held`: there
// are rows in 8 bits.
int hold_args(const char* who, int64_t rows, int64_t cols, int dtype, const void* q,
              int64_t q_stride, const void* scales, HoldArgs* a, int64_t* groups, bool held = true) {
  FMOE_REQUIRE(rows >= 0 && cols >= 1, "%s: bad sizes rows=%lld columns=%lld", who, (long long)rows,
               (long long)cols);
  FMOE_REQUIRE(fmoe_host::is_float_dtype(dtype), "%s: bad dtype %d", who, dtype);
  FMOE_REQUIRE(rows == 0 || !held || (q && scales), "%s: null device pointer", who);
  FMOE_REQUIRE(!held || (reinterpret_cast<uintptr_t>(q) % 16 == 0 && q_stride % 16 == 0 &&
                         q_stride >= fmoe_host::round_up(cols, kHoldBlock)),
               "%s: 8-bit rows must start at multiples of 16 bytes and have room for whole blocks",
               who);
  const int64_t vectors = fmoe_host::round_up(cols, kHoldBlock) / 8;
  a->grid.tx = 4;  // 16 lanes: one block
  while (a->grid.tx < 8 && (1 << a->grid.tx) < vectors) ++a->grid.tx;
  const int64_t chunks = (vectors + (1 << a->grid.tx) - 1) >> a->grid.tx;
  a->grid.step = kGroup >> a->grid.tx;
  a->grid.each = dtype == FMOE_F32 ? hold_rows<float>() : hold_rows<bf16_t>();
  const int64_t rows_of_group = a->grid.step * a->grid.each;
  const int64_t high = (rows + rows_of_group - 1) / rows_of_group;
  // a launch has fewer than 2^32 threads
  if (cols > (int64_t(1) << 30) || rows > (int64_t(1) << 34) ||
      high > ((int64_t(1) << 24) - 1) / chunks) {
    fmoe_host::set_error("%s: rows=%lld columns=%lld too large", who, (long long)rows,
                         (long long)cols);
    return FMOE_ERANGE;
  }
  a->grid.chunks = (int)chunks;
  *groups = high * chunks;
  a->rows = rows;
  a->cols = cols;
  a->blocks = (cols + kHoldBlock - 1) / kHoldBlock;
  a->q = static_cast<uint8_t*>(const_cast<void*>(q));
  a->q_stride = q_stride;
  a->scales = static_cast<float*>(const_cast<void*>(scales));
  return FMOE_OK;
}

// Outputs go past the caches from the size at which the combine's does: 32768 x 2048 in bf16, backward 73.5 us
// and 83, restoring 29.2 and 32.2.  Two 16-byte stores a lane, as fp32's, leave lines that are written in
// two parts: restoring takes 97 us so and 60 through the caches (the backward, which also computes,
// 159 and 170).
int goes_past(const HoldArgs& a, int dtype) {
  return a.rows * a.cols * fmoe_host::dtype_bytes(dtype) >= FMOE_STREAM_OUT_BYTES;
}

template <typename F> void by_float(int dtype, F&& f) {
  if (dtype == FMOE_F32) f(float{});
  else if (dtype == FMOE_BF16) f(bf16_t{});
  else f(f16_t{});
}

}  // namespace

extern "C" int fmoe_compress_rows(const void* d_x, int64_t x_row_stride, int64_t rows, int64_t cols,
                                  int dtype, void* d_q, int64_t q_stride, float* d_scales,
                                  void* d_gelu, void* stream) {
  fmoe_host::clear_error();
  const char* who = "fmoe_compress_rows";
  HoldArgs a{};
  int64_t groups;
  const bool held = d_q || d_scales || !d_gelu;
  if (int rc = hold_args(who, rows, cols, dtype, d_q, q_stride, d_scales, &a, &groups, held)) return rc;
  FMOE_REQUIRE(rows == 0 || d_x, "%s: null device pointer", who);
  FMOE_REQUIRE(x_row_stride >= 0, "%s: negative row stride", who);
  if (rows == 0) return FMOE_OK;
  a.x = d_x;
  a.x_stride = x_row_stride;
  a.out = d_gelu;
  by_float(dtype, [&](auto t) {
    using T = decltype(t);
    hipStream_t s = static_cast<hipStream_t>(stream);
    const dim3 grid((unsigned)groups), group(kGroup);
    if (!held) hipLaunchKernelGGL((k_compress<T, false, true>), grid, group, 0, s, a);
    else if (d_gelu) hipLaunchKernelGGL((k_compress<T, true, true>), grid, group, 0, s, a);
    else hipLaunchKernelGGL((k_compress<T, true, false>), grid, group, 0, s, a);
  });
  return fmoe_host::check_launch(who);
}

extern "C" int fmoe_restore_rows(const void* d_q, int64_t q_stride, const float* d_scales,
                                 int64_t scales_per_row, int64_t rows, int64_t cols, void* d_out,
                                 int dtype, void* stream) {
  fmoe_host::clear_error();
  const char* who = "fmoe_restore_rows";
  HoldArgs a{};
  int64_t groups;
  if (int rc = hold_args(who, rows, cols, dtype, d_q, q_stride, d_scales, &a, &groups)) return rc;
  FMOE_REQUIRE(rows == 0 || d_out, "%s: null device pointer", who);
  FMOE_REQUIRE(scales_per_row == 1 || scales_per_row == a.blocks,
               "%s: %lld scales per row, neither one nor one for each block", who,
               (long long)scales_per_row);
  if (rows == 0) return FMOE_OK;
  a.blocks = scales_per_row;
  a.out = d_out;
  a.past = dtype != FMOE_F32 && goes_past(a, dtype);
  by_float(dtype, [&](auto t) {
    hipLaunchKernelGGL((k_restore<decltype(t)>), dim3((unsigned)groups), dim3(kGroup), 0,
                       static_cast<hipStream_t>(stream), a);
  });
  return fmoe_host::check_launch(who);
}

extern "C" int fmoe_gelu_compressed_backward(const void* d_q, int64_t q_stride,
                                             const float* d_scales, const void* d_grad_a,
                                             int64_t grad_row_stride, int64_t rows, int64_t cols,
                                             int dtype, void* d_again, void* d_grad, void* stream) {
  fmoe_host::clear_error();
  const char* who = "fmoe_gelu_compressed_backward";
  HoldArgs a{};
  int64_t groups;
  if (int rc = hold_args(who, rows, cols, dtype, d_q, q_stride, d_scales, &a, &groups)) return rc;
  FMOE_REQUIRE(rows == 0 || (d_grad_a && d_grad), "%s: null device pointer", who);
  FMOE_REQUIRE(grad_row_stride >= 0, "%s: negative row stride", who);
  if (rows == 0) return FMOE_OK;
  a.x = d_grad_a;
  a.x_stride = grad_row_stride;
  a.out = d_grad;
  a.again = d_again;
  a.past = goes_past(a, dtype);
  by_float(dtype, [&](auto t) {
    hipLaunchKernelGGL((k_gelu_backward<decltype(t)>), dim3((unsigned)groups), dim3(kGroup), 0,
                       static_cast<hipStream_t>(stream), a);
  });
  return fmoe_host::check_launch(who);
}
