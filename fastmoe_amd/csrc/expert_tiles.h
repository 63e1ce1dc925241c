// What the experts' products share: which rows and columns a workgroup has, loads that go to LDS directly, and
// the order of what the waves exchange there.  Args: a kernel's arguments, with x_rows, index, index_dtype, off, E, N,
// rows, out, out_stride and groups_n.
#pragma once

#include "rows8.h"

#include <algorithm>

namespace fmoe {

// A tile of up to BM rows of one expert.  Expert E stands for the rows that belong to none.
struct Tile {
  int64_t expert, row;
  int count;
};

// Lane `lane`'s value, in scalar registers: what hangs on a tile is then the same for the whole wave to
// the compiler too.
__device__ __forceinline__ int64_t lane_value(int64_t v, int lane) {
  const uint32_t lo = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)v, lane);
  const uint32_t hi = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)((uint64_t)v >> 32), lane);
  return (int64_t)((uint64_t)hi << 32 | lo);
}

__device__ __forceinline__ int64_t bounded(int64_t v, int64_t most) {
  return min(max(v, (int64_t)0), most);
}

// The tiles of up to 256 experts from e0 on, four of them in each lane: lo[i] is the first row of the
// lane's i-th expert, n[i] its tiles, incl the tiles up to and with this lane's.  One round of loads
// and a prefix sum over the wave; every wave does it for itself, so there is neither a table in
// memory nor a launch that makes it.  Offsets are held to [0, rows]: no value in them makes a wave
// read or write outside the arrays.
constexpr int kScanExperts = 4 * kWave;
constexpr int kBand = 4;
template <int BM> struct TileScan {
  int64_t lo[5];
  int n[4], incl;
  template <typename Args> __device__ __forceinline__ void load(const Args& a, int64_t e0) {
    const int lane = threadIdx.x & (kWave - 1);
#pragma unroll
    for (int i = 0; i < 5; ++i) {
      const int64_t e = min(e0 + lane * 4 + i, a.E);
      lo[i] = e == 0 ? 0 : bounded(a.off[e], a.rows);
    }
    incl = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {  // beyond E both ends are off[E]: no rows
      n[i] = (int)((max(lo[i + 1] - lo[i], (int64_t)0) + BM - 1) / BM);
      incl += n[i];
    }
#pragma unroll
    for (int d = 1; d < kWave; d *= 2) {
      const int up = __shfl_up(incl, d);
      if (lane >= d) incl += up;
    }
  }
  __device__ __forceinline__ int total() const { return __builtin_amdgcn_readlane(incl, kWave - 1); }
  // Tile `want` of these experts, 0 <= want < total(), and its group of columns.  An expert's tiles go
  // in bands of kBand: the workgroups of a band stand next to each other, columns after columns.
  // False only for offsets that are no offsets, whose tiles may pass what an int counts.
  __device__ __forceinline__ bool find(int want, int64_t e0, int groups_n, Tile* t, int* group) const {
    const int mine = n[0] + n[1] + n[2] + n[3];
    const int at = __ffsll((unsigned long long)__ballot(want < incl)) - 1;
    if (at < 0) return false;
    want -= __builtin_amdgcn_readlane(incl - mine, at);
    if (want < 0) return false;
    int64_t expert = e0 + 4 * at, first = 0, end = 0;
    int of = 0;  // the expert's tiles
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int k = __builtin_amdgcn_readlane(n[i], at);
      if (!of && want < k) {
        of = k;
        expert += i;
        first = lane_value(lo[i], at);
        end = lane_value(lo[i + 1], at);
      }
      if (!of) want -= k;
    }
    if (!of) return false;
    const int band = want / kBand, high = min(kBand, of - band * kBand);
    const int unit = (want % kBand) * groups_n + *group;
    want = band * kBand + unit % high;
    *group = unit / high;
    t->expert = expert;
    t->row = first + (int64_t)want * BM;
    t->count = (int)min((int64_t)BM, end - t->row);
    return true;
  }
};

// Where this workgroup's work lies: a tile of rows and a group of columns.  Workgroups go to the eight
// XCDs in turn (blockIdx % 8); each XCD gets one contiguous eighth of the tiles that there are, columns
// innermost, so that the workgroups that run on it together share rows and weights in its L2.
// False where there is no work: the grid is the most tiles that these sizes can have.
constexpr unsigned kXcds = 8;
template <int BM, typename Args> __device__ __forceinline__ bool place(const Args& a, Tile* t, int* group) {
  TileScan<BM> scan;
  int64_t rest = 0, tiles = (a.rows + BM - 1) / BM;  // rest: first row of no expert
  int first = 0;                                     // tiles of the first chunk of experts
  if (a.off) {
    rest = bounded(a.off[a.E], a.rows);
    tiles = (a.rows - rest + BM - 1) / BM;
    for (int64_t e0 = kScanExperts; e0 < a.E; e0 += kScanExperts) {
      scan.load(a, e0);
      tiles += scan.total();
    }
    scan.load(a, 0);
    first = scan.total();
    tiles += first;
  }
  const unsigned columns = (unsigned)a.groups_n;
  const unsigned work = (unsigned)tiles * columns;  // the host has checked that the grid fits 32 bits
  const unsigned xcd = blockIdx.x % kXcds, turn = blockIdx.x / kXcds;
  const unsigned each = work / kXcds, over = work % kXcds;
  if (turn >= each + (xcd < over ? 1 : 0)) return false;
  const unsigned unit = xcd * each + min(xcd, over) + turn;
  int64_t want = unit / columns;
  *group = (int)(unit % columns);
  if (a.off) {
    if (want < first) return scan.find((int)want, 0, a.groups_n, t, group);
    want -= first;
    for (int64_t e0 = kScanExperts; e0 < a.E; e0 += kScanExperts) {
      scan.load(a, e0);
      if (want < scan.total()) return scan.find((int)want, e0, a.groups_n, t, group);
      want -= scan.total();
    }
  }
  t->expert = a.off ? a.E : 0;
  t->row = rest + want * BM;
  if (t->row >= a.rows) return false;
  t->count = (int)min((int64_t)BM, a.rows - t->row);
  return true;
}

// The row of x that packed row r reads; -1 where its index lies outside x.
template <typename Args> __device__ __forceinline__ int64_t source_row(const Args& a, int64_t r) {
  if (!a.index) return r < a.x_rows ? r : -1;
  const int64_t i = load_index(a.index, a.index_dtype, r);
  return i >= 0 && i < a.x_rows ? i : -1;
}

// Four fp32 values before their rounding to fp16.  The compiler would take the last addition and the rounding as
// one instruction, which is no faster, and whose results are not always the fp32 ones' nearest.
template <typename TO> __device__ __forceinline__ void apart(float* f) {
  if constexpr (std::is_same<TO, f16_t>::value) asm("" : "+v"(f[0]), "+v"(f[1]), "+v"(f[2]), "+v"(f[3]));
}

// Rows of no expert: zeros.
template <typename TO, typename Args>
__device__ __forceinline__ void zero_rows(const Args& a, const Tile& t, int64_t n0, int cols) {
  for (int r = 0; r < t.count; ++r)
    for (int64_t n = n0 + threadIdx.x; n < min(n0 + cols, a.N); n += blockDim.x)
      st1(static_cast<TO*>(a.out) + (t.row + r) * a.out_stride + n, 0.f);
}

#define FMOE_LDS __attribute__((address_space(3)))

template <int CPOL> __device__ __forceinline__ void load_piece(const uint8_t* from, uint8_t* to) {
  __builtin_amdgcn_global_load_lds(reinterpret_cast<const FMOE_GLOBAL uint32_t*>(
                                       reinterpret_cast<uintptr_t>(from)),
                                   (FMOE_LDS uint32_t*)to, 16, 0, CPOL);
}
// All but the youngest `LOADS` loads of this wave have arrived, and all its LDS reads.
template <int LOADS> __device__ __forceinline__ void wait_loads() {
  static_assert(LOADS < 64, "vmcnt has six bits");
  __builtin_amdgcn_s_waitcnt((LOADS & 15) | (LOADS >> 4) << 14 | 0x70);
}
// A barrier alone: __syncthreads would also wait for every load to LDS in flight.  The compiler moves no
// access to memory across it, and wait_loads before it orders what the waves share.
__device__ __forceinline__ void barrier() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}
// Between what a wave's lanes write to LDS and what its other lanes read there: LDS serves a wave in order,
// so no wait is needed, but the compiler, which sees one lane's addresses, must keep that order.
__device__ __forceinline__ void wave_order() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}
template <int KB> __device__ __forceinline__ int swizzle(int row) {
  return KB < 256 ? row / (256 / (KB < 256 ? KB : 256)) % (KB / 16) : row % 16;
}

}  // namespace fmoe

namespace {

// Tiles of `bm` rows that `rows` packed rows of up to `E` experts (and of none) have at most.
inline int64_t most_tiles(int64_t rows, int64_t E, bool grouped, int64_t bm) {
  const int64_t even = (rows + bm - 1) / bm;
  return grouped ? std::min(rows, even + E) : even;
}

// Fills in the groups of `bn` columns; the workgroups of tiles of `bm` rows, or -1 where they are too many.
template <typename Args> int64_t grid_of(const char* who, Args* a, int64_t bm, int64_t bn, int64_t threads) {
  const int64_t tiles = most_tiles(a->rows, a->E, a->off != nullptr, bm);
  a->groups_n = (int)((a->N + bn - 1) / bn);
  if (tiles > ((int64_t(1) << 32) - 1) / (a->groups_n * threads)) {
    fmoe_host::set_error("%s: rows=%lld N=%lld too large", who, (long long)a->rows, (long long)a->N);
    return -1;
  }
  return tiles * a->groups_n;
}

}  // namespace
