// Routing of tokens to experts, forward and backward.  For a token's logits l over E experts:
//
//   score   s = softmax(l) or sigmoid(l), over all experts
//   choice  c = s + bias, where there is a bias or a group's score is a sum; else l, which ranks alike
//   groups  a group's score is its highest c, or the sum of its two highest; the best few groups stay
//   ids     the k highest c of what stays, highest first, the lowest index first among equals
//   weights w = scale * u with u = s[ids], or s[ids] / sum(s[ids])
//
// A choice is a comparison of numbers that may lie next to each other, so s is computed in 64 bits (to
// 2^-36) and rounded to fp32 once; the bias and the sum of two are added in fp32.  Whoever rounds the exact scores to
// fp32 has the same ones but for about four in a million, which lie so near the middle of two fp32 numbers that they
// round to the other one, and makes the same choices unless such a score decides one.  The weights are computed from
// the chosen logits in 64 bits: k of them cost little.  Only the sum under a softmax over all experts is fp32 where no
// scores are compared, to 2^-17 and measured to 2^-20 (in 64 bits 32768 tokens with 64 experts take 8.8 us
// instead of 7.7, with 256 experts 22.5 instead of 18.7).  Masked experts (-inf) have no share, and their choice is their
// bias alone; where all that count are masked, no weight either.  A NaN ranks above every number and makes the weights that
// depend on it NaN.
//
// Backward, with g the weights' gradient and S = sum_j u_j g_j over the chosen:
//   softmax, renormalised   dl_i = scale u_i (g_i - S), the chosen alone
//   sigmoid, renormalised   dl_i = scale u_i (1 - s_i) (g_i - S), the chosen alone
//   softmax                 dl_i = scale s_i (g_i [chosen] - S), every expert
//   sigmoid                 dl_i = scale s_i (1 - s_i) g_i, the chosen alone
// The bias only chooses: it has no gradient.
#include "rows8.h"

#include <algorithm>
#include <cmath>

namespace fmoe {

constexpr int kMaxTopK = 64;

struct RouteArgs {
  const void* logits;
  int64_t stride;  // elements
  int64_t T;
  int dtype;
  const float* bias;  // [E], or null
  int E, k, groups, size, top_groups;  // size: experts of a group
  int group_lanes;                     // lanes that hold a group, a power of two
  int two;                             // a group's score is the sum of its two highest
  int sigmoid, renormalize;
  float scale;
  void* weights;  // [T, k]
  int w_dtype;
  int64_t* ids;   // [T, k]
  float* share;   // [T, k]: u; null where no backward follows
  float* rest;    // [T, k]: 1 - s of a sigmoid; null where not wanted
  float* norm;    // [T, 2]: maximum and 1 / sum of a softmax over all experts; null where not wanted
};

// Numbers as whole numbers that order alike: 0 is below -inf, every NaN on top, and -0 is 0.
__device__ __forceinline__ uint32_t order_key(float f) {
  const uint32_t u = __float_as_uint(f + 0.0f);
  if ((u & 0x7fffffffu) > 0x7f800000u) return 0xffffffffu;
  return u ^ ((uint32_t)((int32_t)u >> 31) | 0x80000000u);
}
__device__ __forceinline__ float key_value(uint32_t key) {
  return __uint_as_float(key & 0x80000000u ? key ^ 0x80000000u : ~key);
}

// e^x to 2^-36 for |x| <= 700 (NaN stays), `about` x in fp32: x = n ln 2 + r with |r| below 0.347, the series of e^r up to r^9, and n
// added to its exponent.  Only what needs 64 bits is in them: rounding, conversions and scaling take two to four times
// as long there as an fp32 instruction.
__device__ __forceinline__ double exp64(double x, float about) {
  const float n = __builtin_rintf(about * 1.44269504f);
  const double r = __builtin_fma((double)n, -0.69314718055994531, x);  // |n| <= 1010: off by 6e-14 at most
  double p = 1.0 / 362880;
  p = __builtin_fma(p, r, 1.0 / 40320);
  p = __builtin_fma(p, r, 1.0 / 5040);
  p = __builtin_fma(p, r, 1.0 / 720);
  p = __builtin_fma(p, r, 1.0 / 120);
  p = __builtin_fma(p, r, 1.0 / 24);
  p = __builtin_fma(p, r, 1.0 / 6);
  p = __builtin_fma(p, r, 0.5);
  p = __builtin_fma(p, r, 1.0);
  p = __builtin_fma(p, r, 1.0);
  const uint64_t u = __builtin_bit_cast(uint64_t, p);
  const uint32_t hi = (uint32_t)(u >> 32) + ((uint32_t)(int)n << 20);
  return __builtin_bit_cast(double, (uint64_t)hi << 32 | (uint32_t)u);
}
__device__ __forceinline__ double exp64(float x) { return exp64((double)x, x); }
// Within +-700, where e^x is neither infinite nor zero; NaN stays.
__device__ __forceinline__ float bounded700(float x) {
  return __builtin_elementwise_maximum(__builtin_elementwise_minimum(x, 700.f), -700.f);
}
// e^(l - from) for l <= from, not below e^-700; NaN stays.
__device__ __forceinline__ double power64(float l, float from) {
  const double d = (double)l - (double)from, bounded = d < -700. ? -700. : d;
  return exp64(bounded, (float)bounded);
}
// 1 / x for a positive normal x, to 2^-40: the hardware's estimate (2^-22 at least) and one step of Newton's.
__device__ __forceinline__ double inverse64(double x) {
  const double y = __builtin_amdgcn_rcp(x);
  return __builtin_fma(__builtin_fma(-x, y, 1.0), y, y);
}
__device__ __forceinline__ double sigmoid64(float l) { return inverse64(1. + exp64(-bounded700(l))); }

// Over the L lanes of a token, as the hardware moves them: a lane's value and its neighbour's, pairs, halves of eight
// (mirrored, where the quads agree already), halves of a row; rows and halves of the wave come as both lanes' values.
struct Both {
  uint32_t a, b;
};
template <int STEP> __device__ __forceinline__ Both across(uint32_t v) {
  if constexpr (STEP == 1) return {v, dpp<0xb1>(v)};
  else if constexpr (STEP == 2) return {v, dpp<0x4e>(v)};
  else if constexpr (STEP == 4) return {v, dpp<0x141>(v)};
  else if constexpr (STEP == 8) return {v, dpp<0x140>(v)};
  else if constexpr (STEP == 16) {
    const auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    return {r[0], r[1]};
  } else {
    const auto r = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    return {r[0], r[1]};
  }
}
struct Both64 {
  double a, b;
};
template <int STEP> __device__ __forceinline__ Both64 across(double v) {
  const uint64_t u = __builtin_bit_cast(uint64_t, v);
  const Both lo = across<STEP>((uint32_t)u), hi = across<STEP>((uint32_t)(u >> 32));
  return {__builtin_bit_cast(double, (uint64_t)hi.a << 32 | lo.a), __builtin_bit_cast(double, (uint64_t)hi.b << 32 | lo.b)};
}
template <int STEP> __device__ __forceinline__ uint32_t step_max(uint32_t v) {
  const Both w = across<STEP>(v);
  return max(w.a, w.b);
}
template <int STEP> __device__ __forceinline__ double step_max(double v) {
  const Both64 w = across<STEP>(v);
  return __builtin_fmax(w.a, w.b);
}
template <int L, typename V> __device__ __forceinline__ V token_max(V v) {
  v = step_max<2>(step_max<1>(v));
  if constexpr (L >= 8) v = step_max<4>(v);
  if constexpr (L >= 16) v = step_max<8>(v);
  if constexpr (L >= 64) v = step_max<32>(step_max<16>(v));
  return v;
}
template <int STEP> __device__ __forceinline__ float step_sum(float v) {
  const Both w = across<STEP>(__float_as_uint(v));
  return __uint_as_float(w.a) + __uint_as_float(w.b);
}
template <int STEP> __device__ __forceinline__ double step_sum(double v) {
  const Both64 w = across<STEP>(v);
  return w.a + w.b;
}
template <int L, typename V> __device__ __forceinline__ V token_sum(V v) {
  v = step_sum<2>(step_sum<1>(v));
  if constexpr (L >= 8) v = step_sum<4>(v);
  if constexpr (L >= 16) v = step_sum<8>(v);
  if constexpr (L >= 64) v = step_sum<32>(step_sum<16>(v));
  return v;
}

// VPL consecutive experts, of which `count` are there; the others read as zero.
template <int VPL, typename T>
__device__ __forceinline__ void load_logits(const T* row, int first, int count, float* v) {
  if constexpr (VPL % 8 == 0) {
#pragma unroll
    for (int i = 0; i < VPL; i += 8)
      Eight<T>::V::cvt(Eight<T>::template load<false>(row, first + i, first + count), v + i);
  } else {
#pragma unroll
    for (int i = 0; i < VPL; ++i) v[i] = i < count ? ld1(row + first + i) : 0.f;
  }
}

// A choice with its expert as one whole number below 2^44, in a double: the largest is the highest choice, of equal ones that of
// the lowest index, and a comparison of two is one instruction.  -1 stands for none.
constexpr int kIndexes = 4096;
__device__ __forceinline__ double ranked(uint32_t key, int index) {
  return __builtin_fma((double)key, (double)kIndexes, (double)(kIndexes - 1 - index));
}
__device__ __forceinline__ int rank_index(double r) {  // r + 2^52 has r in its low bits
  return kIndexes - 1 - (int)(__builtin_bit_cast(uint64_t, r + 4503599627370496.0) & (kIndexes - 1));
}
__device__ __forceinline__ uint32_t rank_key(double r) { return (uint32_t)(r * (1.0 / kIndexes)); }

// Falling order, by Batcher's merges of sorted halves (odd-even merge sort).
template <int N> __device__ __forceinline__ void sort_falling(double* s) {
#pragma unroll
  for (int p = 1; p < N; p *= 2)
#pragma unroll
    for (int k = p; k >= 1; k /= 2)
#pragma unroll
      for (int j = k % p; j + k < N; j += 2 * k)
#pragma unroll
        for (int i = 0; i < k; ++i)
          if (i + j + k < N && (i + j) / (2 * p) == (i + j + k) / (2 * p)) {
            const double x = s[i + j], y = s[i + j + k];
            s[i + j] = __builtin_fmax(x, y);
            s[i + j + k] = __builtin_fmin(x, y);
          }
}

// A token's experts lie in the registers of L lanes, VPL consecutive ones in each (a group starts in a lane of
// its own), so that a wave takes 64 / L tokens and a maximum over them is a few register moves.  Each lane sorts
// its own once; then a round takes the highest of the lanes' first ones, and its lane moves the others up.  (Rounds that searched all
// of a lane's for the highest again took 34 us for 32768 tokens, 256 experts in groups and 8 of them; so 26.6, with the vector
// units two thirds busy: sums, sorts and 64-bit scores bound it, not the 37 MB.)
template <int VPL, int L, bool SCORES> __global__ __launch_bounds__(kGroup) void k_route(RouteArgs a) {
  __shared__ uint16_t chosen[kGroup / L][kMaxTopK];  // where a token's choices pass its lanes
  const int lane = threadIdx.x & (kWave - 1), sub = lane & (L - 1);
  const int slot = threadIdx.x / L;
  const int64_t token = (int64_t)blockIdx.x * (kGroup / L) + slot;
  const int64_t at = min(token, a.T - 1);  // lanes without a token go along with the last one
  const int g = sub / a.group_lanes, part = sub & (a.group_lanes - 1);
  const int first = g < a.groups ? g * a.size + min(part * VPL, a.size) : a.E;
  const int count = g < a.groups ? min(VPL, (g + 1) * a.size - first) : 0;

  float v[VPL];
  if (a.dtype == FMOE_F32) load_logits<VPL>(static_cast<const float*>(a.logits) + at * a.stride, first, count, v);
  else if (a.dtype == FMOE_BF16)
    load_logits<VPL>(static_cast<const bf16_t*>(a.logits) + at * a.stride, first, count, v);
  else load_logits<VPL>(static_cast<const f16_t*>(a.logits) + at * a.stride, first, count, v);
  const bool whole = !a.sigmoid && (SCORES || !a.renormalize);  // the softmax over all experts is wanted
  float top = 0.f;
  bool empty = false;  // every expert is masked
  double inv = 0.;     // 1 / the sum of e^(l - top)
  if (whole) {
    uint32_t high = 0;
#pragma unroll
    for (int i = 0; i < VPL; ++i) high = max(high, i < count ? order_key(v[i]) : 0u);
    top = key_value(token_max<L>(high));
    empty = top == -HUGE_VALF;
    if (empty) top = 0.f;
  }
  auto power = [&](int i) { return i < count && !empty ? power64(v[i], top) : 0.; };
  if (whole) {
    if constexpr (SCORES) {
      double sum = 0.;
#pragma unroll
      for (int i = 0; i < VPL; ++i) sum += power(i);
      inv = empty ? 0. : 1. / token_sum<L>(sum);
    } else {
      float sum = 0.f;
#pragma unroll
      for (int i = 0; i < VPL; ++i) sum += i < count && !empty ? expf(v[i] - top) : 0.f;
      inv = empty ? 0. : 1. / (double)token_sum<L>(sum);
    }
  }
  double s[VPL];
  float bias[SCORES ? VPL : 1];
  if constexpr (SCORES) {
#pragma unroll
    for (int i = 0; i < VPL; ++i) bias[i] = 0.f;
    if (a.bias) load_logits<VPL>(a.bias, first, count, bias);
  }
#pragma unroll
  for (int i = 0; i < VPL; ++i) {
    float c = v[i];
    if constexpr (SCORES) {
      c = a.sigmoid ? (float)sigmoid64(v[i]) : (float)(power(i) * inv);
      if (a.bias) c += bias[i];
    }
    s[i] = i < count ? ranked(order_key(c), first + i) : -1.;
  }
  sort_falling<VPL>(s);

  if (a.top_groups < a.groups) {
    double high = s[0], next = VPL > 1 ? s[VPL > 1 ? 1 : 0] : -1.;
    auto join = [&](auto step) {
      constexpr int kStep = decltype(step)::value;
      if (kStep < L && a.group_lanes > kStep) {
        const Both64 h = across<kStep>(high), n = across<kStep>(next);
        next = __builtin_fmax(__builtin_fmin(h.a, h.b), __builtin_fmax(n.a, n.b));
        high = __builtin_fmax(h.a, h.b);
      }
    };
    join(std::integral_constant<int, 1>{});
    join(std::integral_constant<int, 2>{});
    join(std::integral_constant<int, 4>{});
    join(std::integral_constant<int, 8>{});
    join(std::integral_constant<int, 16>{});
    join(std::integral_constant<int, 32>{});
    double score = -1.;
    if (g < a.groups) {
      uint32_t key = rank_key(high);
      if (a.two && next >= 0.) key = order_key(key_value(key) + key_value(rank_key(next)));
      score = ranked(key, g);
    }
    bool stays = false;
    for (int r = 0; r < a.top_groups; ++r)
      if (score == token_max<L>(score)) {
        stays = true;
        score = -1.;
      }
    if (!stays) s[0] = -1.;  // never the highest
  }

  int mine = 0;  // the choice that this lane has: number `sub`
  auto rounds = [&](auto depth) __attribute__((always_inline)) {
    constexpr int kDepth = decltype(depth)::value;
    for (int r = 0; r < a.k; ++r) {
      const double m = token_max<L>(s[0]);
      const int id = rank_index(m);
      if (a.k > L) {
        if (sub == 0) chosen[slot][r] = (uint16_t)id;
      } else if (sub == r) mine = id;
      const bool won = s[0] == m;
#pragma unroll
      for (int i = 0; i < kDepth; ++i) {
        const double up = i + 1 < VPL ? s[i + 1 < VPL ? i + 1 : 0] : -1.;
        s[i] = won ? up : s[i];
      }
    }
  };
  if (VPL > 8 && a.k <= 8) rounds(std::integral_constant<int, VPL < 8 ? VPL : 8>{});
  else rounds(std::integral_constant<int, VPL>{});
  if (a.k > L) {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");  // a wave's LDS accesses are served in order
    __builtin_amdgcn_wave_barrier();
    mine = sub < a.k ? chosen[slot][sub] : 0;
  }

  auto logit = [&](int id) {
    const int64_t i = at * a.stride + id;
    return load_weight(a.logits, a.dtype, i);
  };
  // lane `sub` has the choices sub, sub + L, ...; most tokens have no more than L
  const float mine_l = logit(mine);
  auto each = [&](auto&& f) {
    if (sub < a.k) f(sub, mine, mine_l);
    for (int j = sub + L; j < a.k; j += L) f(j, (int)chosen[slot][j], logit(chosen[slot][j]));
  };
  float from = top;  // u = e^(l - from) * over, for a sigmoid divided by 1 + e^l too
  double over = inv;
  bool none = empty;
  auto unit = [&](float l) {
    if (!a.sigmoid) return power64(l, from);
    const double e = exp64(-__builtin_fabsf(bounded700(l)));  // e^-|l|
    double n = l > 0.f ? 1. : e;
    if (from != 0.f) n = power64(l, from);
    return n * inverse64(1. + e);
  };
  if (a.renormalize) {
    uint32_t high = 0;
    each([&](int, int, float l) { high = max(high, order_key(l)); });
    const float m = key_value(token_max<L>(high));
    none = m == -HUGE_VALF;
    from = none || (a.sigmoid && m > 0.f) ? 0.f : m;
    double sum = 0.;
    each([&](int, int, float l) { sum += l == -HUGE_VALF ? 0. : unit(l); });
    over = 1. / token_sum<L>(sum);
  } else if (a.sigmoid) {
    from = 0.f;
    over = 1.;
  }
  if (token >= a.T) return;
  each([&](int j, int id, float l) {
    const int64_t i = token * a.k + j;
    const double u = none || l == -HUGE_VALF ? 0. : unit(l) * over;
    a.ids[i] = id;
    const float w = (float)(u * (double)a.scale);
    if (a.w_dtype == FMOE_F32) static_cast<float*>(a.weights)[i] = w;
    else if (a.w_dtype == FMOE_BF16) st1(static_cast<bf16_t*>(a.weights) + i, w);
    else st1(static_cast<f16_t*>(a.weights) + i, w);
    if (a.share) a.share[i] = (float)u;
    if (a.rest) a.rest[i] = (float)sigmoid64(-l);
  });
  if (a.norm && sub == 0) {
    a.norm[2 * token] = top;
    a.norm[2 * token + 1] = (float)inv;
  }
}

struct RouteBwdArgs {
  const void* grad;  // [T, k]
  int grad_dtype;
  const int64_t* ids;
  const float *share, *rest, *norm;  // norm: the softmax over all experts, else null
  const void* logits;                // read with norm
  int64_t stride, T;
  int E, k, lanes;  // lanes of a token, a power of two
  int renormalize;
  float scale;
  void* out;  // [T, E]
};

// Eight columns of a token's row in a lane at a time, each row written once.  Every lane reads the token's k
// gradients itself: they come from the cache, and no lane waits for another.  32768 tokens,
// 6 of 64 experts, bf16, take 8 us, half of it a launch's.
template <typename T> __global__ __launch_bounds__(kGroup) void k_route_bwd(RouteBwdArgs a) {
  const int64_t token = ((int64_t)blockIdx.x * kGroup + threadIdx.x) / a.lanes;
  const int sub = threadIdx.x & (a.lanes - 1);
  if (token >= a.T) return;
  const int64_t base = token * a.k;
  float dot = 0.f;
  if (a.renormalize || a.norm)
    for (int j = 0; j < a.k; ++j)
      dot = __builtin_fmaf(a.share[base + j], load_weight(a.grad, a.grad_dtype, base + j), dot);
  const float top = a.norm ? a.norm[2 * token] : 0.f, inv = a.norm ? a.norm[2 * token + 1] : 0.f;
  for (int c = sub * 8; c < a.E; c += a.lanes * 8) {
    float f[8];
    if (a.norm) {
      Eight<T>::V::cvt(Eight<T>::template load<false>(static_cast<const T*>(a.logits) + token * a.stride, c, a.E), f);
#pragma unroll
      for (int i = 0; i < 8; ++i) f[i] = expf(f[i] - top) * inv * -dot;
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) f[i] = 0.f;
    }
#pragma unroll 4
    for (int j = 0; j < a.k; ++j) {
      const float g = load_weight(a.grad, a.grad_dtype, base + j);
      float d = a.share[base + j] * (a.renormalize ? g - dot : g);
      if (a.rest) d *= a.rest[base + j];
      const int place = (int)a.ids[base + j] - c;
#pragma unroll
      for (int i = 0; i < 8; ++i) f[i] += place == i ? d : 0.f;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] *= a.scale;
    Eight<T>::store(static_cast<T*>(a.out) + token * a.E, c, a.E, Eight<T>::V::pack(f));
  }
}

}  // namespace fmoe

using namespace fmoe;

namespace {

constexpr int64_t kMaxExperts = 4096, kMaxGrouped = 1024, kMaxGroups = 64;

int power_of_two(int n) {
  int p = 1;
  while (p < n) p *= 2;
  return p;
}

template <int VPL, int L> void launch_route(const RouteArgs& a, bool scores, hipStream_t s) {
  const dim3 grid((unsigned)((a.T + kGroup / L - 1) / (kGroup / L)));
  if (scores) hipLaunchKernelGGL((k_route<VPL, L, true>), grid, dim3(kGroup), 0, s, a);
  else hipLaunchKernelGGL((k_route<VPL, L, false>), grid, dim3(kGroup), 0, s, a);
}

int check_route(const char* who, int64_t T, int64_t E, int64_t k, int dtype, int w_dtype) {
  FMOE_REQUIRE(T >= 0 && E >= 1 && k >= 1 && k <= E, "%s: bad sizes tokens=%lld experts=%lld top_k=%lld", who,
               (long long)T, (long long)E, (long long)k);
  FMOE_REQUIRE(fmoe_host::is_float_dtype(dtype) && fmoe_host::is_float_dtype(w_dtype), "%s: bad dtype %d or %d",
               who, dtype, w_dtype);
  if (E > kMaxExperts || k > kMaxTopK || T > (int64_t(1) << 25)) {
    fmoe_host::set_error("%s: tokens=%lld experts=%lld top_k=%lld too large", who, (long long)T, (long long)E,
                         (long long)k);
    return FMOE_ERANGE;
  }
  return FMOE_OK;
}

}  // namespace

extern "C" int fmoe_route(const void* d_logits, int64_t row_stride, int64_t num_tokens, int64_t num_experts,
                          int dtype, const float* d_bias, int64_t top_k, int score, int64_t groups,
                          int64_t top_groups, int group_score, int renormalize, float scale, void* d_weights,
                          int weight_dtype, int64_t* d_ids, float* d_share, float* d_rest, float* d_norm,
                          void* stream) {
  fmoe_host::clear_error();
  const char* who = "fmoe_route";
  const int64_t T = num_tokens, E = num_experts;
  if (int rc = check_route(who, T, E, top_k, dtype, weight_dtype)) return rc;
  FMOE_REQUIRE(score == FMOE_SCORE_SOFTMAX || score == FMOE_SCORE_SIGMOID, "%s: bad score %d", who, score);
  FMOE_REQUIRE(group_score == FMOE_GROUP_MAX || group_score == FMOE_GROUP_TOP2, "%s: bad group score %d", who,
               group_score);
  FMOE_REQUIRE(groups >= 1 && groups <= E && E % groups == 0 && top_groups >= 1 && top_groups <= groups,
               "%s: %lld of %lld groups of %lld experts", who, (long long)top_groups, (long long)groups, (long long)E);
  FMOE_REQUIRE(top_k <= top_groups * (E / groups), "%s: top_k=%lld of %lld experts", who, (long long)top_k,
               (long long)(top_groups * (E / groups)));
  if (groups > 1 && (E > kMaxGrouped || groups > kMaxGroups)) {
    fmoe_host::set_error("%s: %lld groups of %lld experts too large", who, (long long)groups, (long long)E);
    return FMOE_ERANGE;
  }
  FMOE_REQUIRE(row_stride >= 0, "%s: negative row stride", who);
  FMOE_REQUIRE(std::isfinite(scale), "%s: the scale is not a finite fp32 number", who);
  if (T == 0) return FMOE_OK;
  FMOE_REQUIRE(d_logits && d_weights && d_ids, "%s: null device pointer", who);
  const bool scores = d_bias || (groups > 1 && group_score == FMOE_GROUP_TOP2);
  if (top_groups == groups) groups = top_groups = 1;  // all stay
  RouteArgs a{d_logits, row_stride, T, dtype, d_bias, (int)E, (int)top_k, (int)groups, (int)(E / groups),
              (int)top_groups, 1, group_score == FMOE_GROUP_TOP2, score == FMOE_SCORE_SIGMOID, renormalize != 0,
              scale, d_weights, weight_dtype, d_ids, d_share, d_rest, d_norm};
  // the lanes that hold a token's groups, with `vpl` experts in each
  auto lanes = [&](int vpl) {
    a.group_lanes = power_of_two((a.size + vpl - 1) / vpl);
    return a.group_lanes * a.groups;
  };
  hipStream_t s = static_cast<hipStream_t>(stream);
  // Four experts in a lane make short waves, sixteen fewer of them: 256 experts in 8 groups take 5.6 us instead of 6.8 with 8
  // tokens, 7.4 instead of 7.6 with 2048, 10.4 instead of 7.7 with 4096; 64 experts 3.5 instead of 5.4 with 8 tokens, 4.4
  // instead of 5.9 with 8192, 5.6 instead of 6.1 with 16384.  128 experts would leave half of the lanes idle: 4.3 instead of
  // 4.3 with 8 tokens, 5.4 instead of 4.8 with 2048.
  const int few = lanes(4), few_l = few <= 16 ? 16 : 64;
  if ((few <= 16 || few == 64) && T * few_l <= (1 << 17)) {
    if (few <= 16) launch_route<4, 16>(a, scores, s);
    else launch_route<4, 64>(a, scores, s);
  } else if (lanes(16) <= 4) launch_route<16, 4>(a, scores, s);
  else if (lanes(16) <= 16) launch_route<16, 16>(a, scores, s);
  else if (lanes(16) <= 64) launch_route<16, 64>(a, scores, s);
  else {
    // Above 1024 experts (or as many in groups that leave lanes idle) a lane holds 64 and a SIMD one wave: 2048 tokens' 8 of
    // 4096 take 18 us by their logits, with a bias 42 (sigmoid) and 59 (softmax), bound by 64-bit scores; 64 of them 161 us,
    // as many rounds one after the other.
    lanes(64);
    launch_route<64, 64>(a, scores, s);
  }
  return fmoe_host::check_launch(who);
}

extern "C" int fmoe_route_backward(const void* d_grad, int grad_dtype, const int64_t* d_ids, const float* d_share,
                                   const float* d_rest, const float* d_norm, const void* d_logits,
                                   int64_t row_stride, int64_t num_tokens, int64_t num_experts, int64_t top_k,
                                   int dtype, int renormalize, float scale, void* d_grad_logits, void* stream) {
  fmoe_host::clear_error();
  const char* who = "fmoe_route_backward";
  const int64_t T = num_tokens, E = num_experts;
  if (int rc = check_route(who, T, E, top_k, dtype, grad_dtype)) return rc;
  FMOE_REQUIRE(row_stride >= 0, "%s: negative row stride", who);
  FMOE_REQUIRE(!d_norm || (!renormalize && !d_rest), "%s: a softmax over all experts is not renormalised", who);
  if (T == 0) return FMOE_OK;
  FMOE_REQUIRE(d_grad && d_ids && d_share && d_grad_logits && (!d_norm || d_logits), "%s: null device pointer", who);
  const int lanes = std::min(kWave, power_of_two((int)((E + 7) / 8)));
  const RouteBwdArgs a{d_grad, grad_dtype, d_ids, d_share, d_rest, d_norm, d_logits, row_stride, T, (int)E,
                       (int)top_k, lanes, renormalize != 0, scale, d_grad_logits};
  const dim3 grid((unsigned)((T * lanes + kGroup - 1) / kGroup));
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (dtype == FMOE_F32) hipLaunchKernelGGL((k_route_bwd<float>), grid, dim3(kGroup), 0, s, a);
  else if (dtype == FMOE_BF16) hipLaunchKernelGGL((k_route_bwd<bf16_t>), grid, dim3(kGroup), 0, s, a);
  else hipLaunchKernelGGL((k_route_bwd<f16_t>), grid, dim3(kGroup), 0, s, a);
  return fmoe_host::check_launch(who);
}
