// Routing of tokens to experts, forward and backward.  For a token's logits l over E experts:
//
//   score   s = softmax(l) or sigmoid(l), over all experts
//   choice  c = s + bias, where there is a bias or a group's score is a sum; else l, which ranks alike
//   groups  a group's score is its highest c, or the sum of its two highest; the best few groups stay
//   ids     the k highest c of what stays, highest first, the lowest index first among equals
//   weights w = scale * u with u = s[ids], or s[ids] / sum(s[ids])
//
// A choice is a comparison of numbers that may lie next to each other, so s is computed in 64 bits (to
// 2^-36) and rounded to fp32 once; the bias and the sum of two are added in fp32.  Whoever rounds the same
// scores to fp32 makes the same choices.  The weights are computed from the chosen logits in 64 bits: k of
// them cost little.  Masked experts (-inf) have no share; where all that count are masked, no weight either.
// A NaN ranks above every number and makes the weights that depend on it NaN.
//
// Backward, with g the weights' gradient and S = sum_j u_j g_j over the chosen:
//   softmax, renormalised   dl_i = scale u_i (g_i - S), the chosen alone
//   sigmoid, renormalised   dl_i = scale u_i (1 - s_i) (g_i - S), the chosen alone
//   softmax                 dl_i = scale s_i (g_i [chosen] - S), every expert
//   sigmoid                 dl_i = scale s_i (1 - s_i) g_i, the chosen alone
// The bias only chooses: it has no gradient.
#include "rows8.h"

#include <algorithm>

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

// e^x to 2^-36 for any x (NaN stays): x = n ln 2 + r, |r| <= ln 2 / 2, and the series of e^r up to r^9.
__device__ __forceinline__ double exp64(double x) {
  x = x < -700.0 ? -700.0 : x > 700.0 ? 700.0 : x;
  const double n = __builtin_rint(x * 1.4426950408889634);
  const double r = __builtin_fma(n, -0.69314718055994531, x);  // |n| <= 1010: off by 6e-14 at most
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
  return __builtin_ldexp(p, (int)n);
}
// 1 / x for a positive normal x: the hardware's estimate and two steps of Newton's.
__device__ __forceinline__ double inverse64(double x) {
  double y = __builtin_amdgcn_rcp(x);
  y = __builtin_fma(__builtin_fma(-x, y, 1.0), y, y);
  return __builtin_fma(__builtin_fma(-x, y, 1.0), y, y);
}

// Over the L lanes of a token, L and the lanes' order as the hardware moves them: neighbours, pairs, halves
// of eight (mirrored, where the quads agree already), halves of a row, rows.
template <int STEP, typename F> __device__ __forceinline__ uint32_t across(uint32_t v, F&& f) {
  if constexpr (STEP == 1) return f(v, dpp<0xb1>(v));
  else if constexpr (STEP == 2) return f(v, dpp<0x4e>(v));
  else if constexpr (STEP == 4) return f(v, dpp<0x141>(v));
  else if constexpr (STEP == 8) return f(v, dpp<0x140>(v));
  else return f(v, (uint32_t)__shfl_xor((int)v, STEP));
}
template <int L> __device__ __forceinline__ uint32_t token_max(uint32_t v) {
  auto most = [](uint32_t a, uint32_t b) { return max(a, b); };
  v = across<1>(v, most);
  v = across<2>(v, most);
  if constexpr (L >= 16) v = across<8>(across<4>(v, most), most);
  if constexpr (L >= 64) v = across<32>(across<16>(v, most), most);
  return v;
}
template <int L, typename V> __device__ __forceinline__ V token_sum(V v) {
#pragma unroll
  for (int d = 1; d < L; d *= 2) v += __shfl_xor(v, d);
  return v;
}
// The lanes of this token for which `p` holds, lane 0 of them in bit 0.
template <int L> __device__ __forceinline__ uint64_t token_ballot(bool p, int lane) {
  const uint64_t b = __ballot(p);
  if constexpr (L == kWave) return b;
  else return b >> (lane & ~(L - 1)) & ((uint64_t(1) << L) - 1);
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

// A token's experts lie in the registers of L lanes, VPL consecutive ones in each (a group starts in a lane of
// its own), so that a wave takes 64 / L tokens and a maximum over them is a few register moves.
template <int VPL, int L, bool SCORES> __global__ __launch_bounds__(kGroup) void k_route(RouteArgs a) {
  __shared__ uint16_t chosen[kGroup / L][kMaxTopK];
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
  uint32_t key[VPL], best = 0;
#pragma unroll
  for (int i = 0; i < VPL; ++i) {
    key[i] = i < count ? order_key(v[i]) : 0;
    best = max(best, key[i]);
  }
  const bool whole = !a.sigmoid && (SCORES || !a.renormalize);  // the softmax over all experts is wanted
  float top = 0.f;
  bool empty = false;  // every expert is masked
  double inv = 0.;     // 1 / the sum of e^(l - top)
  if (whole) {
    top = key_value(token_max<L>(best));
    empty = top == -HUGE_VALF;
    if (empty) top = 0.f;
  }
  if constexpr (SCORES) {
    double e[VPL <= 16 ? VPL : 1];
    auto power = [&](int i) { return i < count && !empty ? exp64((double)v[i] - (double)top) : 0.; };
    if (whole) {
      double sum = 0.;
#pragma unroll
      for (int i = 0; i < VPL; ++i) {
        const double p = power(i);
        if constexpr (VPL <= 16) e[i] = p;
        sum += p;
      }
      sum = token_sum<L>(sum);
      inv = empty ? 0. : 1. / sum;
    }
    best = 0;
#pragma unroll
    for (int i = 0; i < VPL; ++i) {
      if (i < count) {
        float s;
        if (a.sigmoid) s = (float)inverse64(1. + exp64(-(double)v[i]));
        else if constexpr (VPL <= 16) s = (float)(e[i] * inv);
        else s = (float)(power(i) * inv);
        key[i] = order_key(a.bias ? s + a.bias[first + i] : s);
      }
      best = max(best, key[i]);
    }
  } else if (whole) {
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < VPL; ++i) sum += i < count && !empty ? expf(v[i] - top) : 0.f;
    sum = token_sum<L>(sum);
    inv = empty ? 0. : 1. / (double)sum;
  }

  if (a.top_groups < a.groups) {
    uint32_t high = best, next = 0;
    if (a.two) {
      bool seen = false;  // the highest once, the others compete for the second place
#pragma unroll
      for (int i = 0; i < VPL; ++i) {
        const bool it = key[i] == high && !seen;
        seen |= it;
        next = max(next, it ? 0u : key[i]);
      }
    }
    auto join = [&](auto step) {
      constexpr int kStep = decltype(step)::value;
      if (kStep < L && a.group_lanes > kStep) {
        auto other = [](uint32_t, uint32_t q) { return q; };
        const uint32_t h = across<kStep>(high, other), n = across<kStep>(next, other);
        next = max(min(high, h), max(next, n));
        high = max(high, h);
      }
    };
    join(std::integral_constant<int, 1>{});
    join(std::integral_constant<int, 2>{});
    join(std::integral_constant<int, 4>{});
    join(std::integral_constant<int, 8>{});
    join(std::integral_constant<int, 16>{});
    join(std::integral_constant<int, 32>{});
    uint32_t score = g < a.groups ? high : 0;
    if (a.two && next) score = order_key(key_value(high) + key_value(next));
    bool stays = false;
    for (int r = 0; r < a.top_groups; ++r) {
      const uint32_t m = token_max<L>(score);
      const int winner = __ffsll((unsigned long long)token_ballot<L>(score == m, lane)) - 1;
      if (winner / a.group_lanes == g) {
        stays = true;
        score = 0;
      }
    }
    if (!stays) {
#pragma unroll
      for (int i = 0; i < VPL; ++i) key[i] = 0;
      best = 0;
    }
  }

  for (int r = 0; r < a.k; ++r) {
    const uint32_t m = token_max<L>(best);
    const int winner = __ffsll((unsigned long long)token_ballot<L>(best == m, lane)) - 1;
    if (sub == winner) {
      int it = 0;
#pragma unroll
      for (int i = VPL - 1; i >= 0; --i) it = key[i] == m ? i : it;
      best = 0;
#pragma unroll
      for (int i = 0; i < VPL; ++i) {
        key[i] = i == it ? 0u : key[i];
        best = max(best, key[i]);
      }
      chosen[slot][r] = (uint16_t)(first + it);
    }
  }
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");  // a wave's LDS accesses are served in order
  __builtin_amdgcn_wave_barrier();

  auto logit = [&](int id) {
    const int64_t i = at * a.stride + id;
    return load_weight(a.logits, a.dtype, i);
  };
  // lane `sub` has the chosen sub, sub + L, ...; most tokens have no more than L
  const int mine = sub < a.k ? chosen[slot][sub] : 0;
  const float mine_l = logit(mine);
  auto each = [&](auto&& f) {
    if (sub < a.k) f(sub, mine, mine_l);
    for (int j = sub + L; j < a.k; j += L) f(j, (int)chosen[slot][j], logit(chosen[slot][j]));
  };
  double from = (double)top, over = inv;  // u = e^(l - from) * over, for a sigmoid divided by 1 + e^l too
  bool none = empty;
  auto unit = [&](float l) {
    if (!a.sigmoid) return exp64((double)l - from);
    if (l > 0.f) return inverse64(1. + exp64(-(double)l));
    return exp64((double)l - from) * inverse64(1. + exp64((double)l));
  };
  if (a.renormalize) {
    uint32_t high = 0;
    each([&](int, int, float l) { high = max(high, order_key(l)); });
    const float m = key_value(token_max<L>(high));
    none = m == -HUGE_VALF;
    from = none ? 0. : a.sigmoid && m > 0.f ? 0. : (double)m;
    double sum = 0.;
    each([&](int, int, float l) { sum += l == -HUGE_VALF ? 0. : unit(l); });
    over = 1. / token_sum<L>(sum);
  } else if (a.sigmoid) {
    from = 0.;
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
    if (a.rest) a.rest[i] = (float)inverse64(1. + exp64((double)l));
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
// gradients itself: they come from the cache, and no lane waits for another.
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
  if (T <= 4096 && lanes(4) <= 64) {
    if (lanes(4) <= 16) launch_route<4, 16>(a, scores, s);
    else launch_route<4, 64>(a, scores, s);
  } else if (lanes(16) <= 4) launch_route<16, 4>(a, scores, s);
  else if (lanes(16) <= 16) launch_route<16, 16>(a, scores, s);
  else if (lanes(16) <= 64) launch_route<16, 64>(a, scores, s);
  else {
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
