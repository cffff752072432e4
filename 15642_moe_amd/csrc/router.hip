// General expert router and its gradient (route.hip holds the layer's own fixed one).
//
//   s_e = sigmoid(x_e)  or  softmax(x)_e         exponentials in 64 bits, rounded to 32
//   v_e = s_e + bias_e                           what the picks are made by
//   group score = sum of the group's one or two largest v; the best groups stay
//   picks = the top_k largest v of those, ties to the lower index
//   w_k = s_k / (sum s + 1e-20) * scale   or   s_k * scale
//
// An expert whose logit or v is -inf or NaN is closed: it is never picked (its
// softmax score is 0).  Slots that no open expert fills hold id -1, weight 0.
// The picks follow from comparisons of 32-bit values, so the 64-bit exponential
// (about 50 f64 operations, which this GPU issues at the f32 rate) is what makes
// them the same on every machine that rounds it once.
//
// Gradient of the weights, with p = s over the picks and P = sum p + 1e-20:
//   ds_k = scale * (g_k - sum_j g_j p_j / P) / P   or   scale * g_k
//   sigmoid: dx_k = ds_k s_k (1 - s_k), zero for experts not picked
//   softmax: dx_e = s_e * (ds_e [picked] - sum_j ds_j p_j)
// The bias balances the experts' load and takes no gradient: the picks are
// piecewise constant in it.
#include "common.h"
#include "launch.h"

#include <math.h>

#include <type_traits>

namespace moe {
namespace {

constexpr int WAVES = 4;  // waves (tokens) per workgroup

template <int DT>
__device__ __forceinline__ float load_as_f32(const void* base, size_t i) {
  if constexpr (DT == DT_F32) return static_cast<const float*>(base)[i];
  else if constexpr (DT == DT_BF16) return __uint_as_float((uint32_t)static_cast<const uint16_t*>(base)[i] << 16);
  else return (float)static_cast<const _Float16*>(base)[i];
}

template <int DT>
__device__ __forceinline__ void store_f32_as(void* base, size_t i, float v) {
  if constexpr (DT == DT_F32) static_cast<float*>(base)[i] = v;
  else if constexpr (DT == DT_BF16) static_cast<uint16_t*>(base)[i] = v == v ? bf16_rne(v) : (uint16_t)0x7FC0;
  else static_cast<_Float16*>(base)[i] = (_Float16)v;
}

// Order-preserving map to uint32; 0 (below every open expert's) for -inf and NaN.
__device__ __forceinline__ uint32_t open_key(float v) {
  if (!(v > -INFINITY)) return 0u;
  v += 0.0f;  // -0 and +0 are equal
  const uint32_t b = __float_as_uint(v);
  return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}

// Reductions over the wave, uniform results: within rows of 16 lanes by DPP moves (lanes
// l ^ 1, l ^ 2, l ^ 7, l ^ 15: no LDS round trip), over the rows by readlane.
constexpr int DPP_XOR1 = 0xB1, DPP_XOR2 = 0x4E, DPP_HALF_MIRROR = 0x141, DPP_MIRROR = 0x140;
template <int CTRL>
__device__ __forceinline__ int dpp(int x) {
  return __builtin_amdgcn_update_dpp(x, x, CTRL, 0xF, 0xF, false);
}
template <int CTRL>
__device__ __forceinline__ float dpp(float x) {
  return __int_as_float(dpp<CTRL>(__float_as_int(x)));
}
template <int CTRL>
__device__ __forceinline__ double dpp(double x) {
  return __hiloint2double(dpp<CTRL>(__double2hiint(x)), dpp<CTRL>(__double2loint(x)));
}
__device__ __forceinline__ uint32_t lane_of(uint32_t x, int l) {
  return (uint32_t)__builtin_amdgcn_readlane((int)x, l);
}
__device__ __forceinline__ float lane_of(float x, int l) {
  return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(x), l));
}
__device__ __forceinline__ double lane_of(double x, int l) {
  return __hiloint2double(__builtin_amdgcn_readlane(__double2hiint(x), l),
                          __builtin_amdgcn_readlane(__double2loint(x), l));
}
// The identity 0 as the old value lets each move and its maximum be one instruction.
template <int CTRL>
__device__ __forceinline__ uint32_t dpp_max(uint32_t x) {
  return max(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, CTRL, 0xF, 0xF, false));
}
__device__ __forceinline__ uint32_t wave_max(uint32_t x) {
  x = dpp_max<DPP_MIRROR>(dpp_max<DPP_HALF_MIRROR>(dpp_max<DPP_XOR2>(dpp_max<DPP_XOR1>(x))));
  return max(max(lane_of(x, 0), lane_of(x, 16)), max(lane_of(x, 32), lane_of(x, 48)));
}
__device__ __forceinline__ float wave_max(float x) {
  x = fmaxf(x, dpp<DPP_XOR1>(x));
  x = fmaxf(x, dpp<DPP_XOR2>(x));
  x = fmaxf(x, dpp<DPP_HALF_MIRROR>(x));
  x = fmaxf(x, dpp<DPP_MIRROR>(x));
  return fmaxf(fmaxf(lane_of(x, 0), lane_of(x, 16)), fmaxf(lane_of(x, 32), lane_of(x, 48)));
}
template <class F>
__device__ __forceinline__ F wave_sum(F x) {
  x += dpp<DPP_XOR1>(x);
  x += dpp<DPP_XOR2>(x);
  x += dpp<DPP_HALF_MIRROR>(x);
  x += dpp<DPP_MIRROR>(x);
  return (lane_of(x, 0) + lane_of(x, 16)) + (lane_of(x, 32) + lane_of(x, 48));
}

// exp(x - m) of a softmax; the maximum's own is 1, also where it is +inf.
template <class F>
__device__ __forceinline__ F exp_below(float x, float m) {
  return x == m ? (F)1 : (F)exp((F)x - (F)m);
}

// One wave per token; lane l holds experts EPL*l .. +EPL.
template <int EPL, int DT, bool SOFTMAX>
__global__ void __launch_bounds__(64 * WAVES)
route_topk_kernel(const void* __restrict__ logits, size_t row_stride, const float* __restrict__ bias, int T, int E,
                  int k, int n_group, int lanes_per_group, int topk_group, int group_top, int renormalize, float scale,
                  float* __restrict__ weights, int32_t* __restrict__ ids) {
  __shared__ float s_v[WAVES][64 * EPL];
  __shared__ float s_sel[WAVES][64];
  __shared__ int s_id[WAVES][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int t = blockIdx.x * WAVES + wave;
  const bool active = t < T;  // idle waves still reach the barriers
  const size_t row = (size_t)(active ? t : T - 1) * row_stride;
  float x[EPL], s[EPL], v[EPL];
#pragma unroll
  for (int j = 0; j < EPL; ++j) {
    const int e = lane * EPL + j;
    x[j] = e < E ? load_as_f32<DT>(logits, row + e) : -INFINITY;
  }
  if constexpr (SOFTMAX) {
    float m = -INFINITY;
#pragma unroll
    for (int j = 0; j < EPL; ++j) m = fmaxf(m, x[j]);
    m = wave_max(m);
    double ex[EPL], sum = 0.0;
#pragma unroll
    for (int j = 0; j < EPL; ++j) {
      ex[j] = x[j] > -INFINITY ? exp_below<double>(x[j], m) : 0.0;
      sum += ex[j];
    }
    sum = wave_sum(sum);
#pragma unroll
    for (int j = 0; j < EPL; ++j) s[j] = sum > 0.0 ? (float)(ex[j] / sum) : 0.0f;
  } else {
#pragma unroll
    for (int j = 0; j < EPL; ++j) {
      const float e = (float)exp(-(double)x[j]);
      s[j] = __fdiv_rn(1.0f, 1.0f + e);
    }
  }
#pragma unroll
  for (int j = 0; j < EPL; ++j) {
    const int e = lane * EPL + j;
    v[j] = x[j] > -INFINITY ? (bias ? s[j] + bias[e] : s[j]) : -INFINITY;
    if (!(v[j] > -INFINITY)) v[j] = -INFINITY;
  }

  uint32_t key[EPL];
#pragma unroll
  for (int j = 0; j < EPL; ++j) key[j] = open_key(v[j]);
  if (n_group > 1) {
    const int gs = E / n_group;
    float m1 = -INFINITY, m2 = -INFINITY;
    auto score = [&] {  // a closed second place adds nothing
      return open_key((group_top == 2 && m2 > -INFINITY) ? m1 + m2 : m1);
    };
    auto add = [&](float y) {
      m2 = fmaxf(m2, fminf(m1, y));
      m1 = fmaxf(m1, y);
    };
    auto merge = [&](float o1, float o2) {
      m2 = fmaxf(fminf(m1, o1), fmaxf(m2, o2));
      m1 = fmaxf(m1, o1);
    };
    if (lanes_per_group > 0) {
      // A group is a power of two of whole lanes, at most a row's 16: its lanes merge
      // their two largest by DPP moves.
#pragma unroll
      for (int j = 0; j < EPL; ++j) add(v[j]);
      if (lanes_per_group > 1) merge(dpp<DPP_XOR1>(m1), dpp<DPP_XOR1>(m2));
      if (lanes_per_group > 2) merge(dpp<DPP_XOR2>(m1), dpp<DPP_XOR2>(m2));
      if (lanes_per_group > 4) merge(dpp<DPP_HALF_MIRROR>(m1), dpp<DPP_HALF_MIRROR>(m2));
      if (lanes_per_group > 8) merge(dpp<DPP_MIRROR>(m1), dpp<DPP_MIRROR>(m2));
      const uint32_t gkey = score();
      const int mine = lane / lanes_per_group;
      int rank = 0;
      for (int g = 0; g < n_group; ++g) {
        const uint32_t o = lane_of(gkey, g * lanes_per_group);
        rank += (o > gkey || (o == gkey && g < mine)) ? 1 : 0;
      }
      if (rank >= topk_group || mine >= n_group) {
#pragma unroll
        for (int j = 0; j < EPL; ++j) key[j] = 0u;
      }
    } else {
      // Lane g scores group g from LDS.
#pragma unroll
      for (int j = 0; j < EPL; ++j) s_v[wave][lane * EPL + j] = v[j];
      __syncthreads();
      if (lane < n_group)
        for (int i = 0; i < gs; ++i) add(s_v[wave][lane * gs + i]);
      const uint32_t gkey = score();
      int rank = 0;
      for (int g = 0; g < n_group; ++g) {
        const uint32_t o = lane_of(gkey, g);
        rank += (o > gkey || (o == gkey && g < lane)) ? 1 : 0;
      }
      const uint64_t kept = __ballot(lane < n_group && rank < topk_group);
#pragma unroll
      for (int j = 0; j < EPL; ++j) {
        const int e = lane * EPL + j;
        if (e >= E || !((kept >> (e / gs)) & 1u)) key[j] = 0u;
      }
    }
  }

  bool sel[EPL];
#pragma unroll
  for (int j = 0; j < EPL; ++j) sel[j] = false;
  int n_sel = 0;
  for (int r = 0; r < k; ++r) {
    uint32_t mine = key[0];
#pragma unroll
    for (int j = 1; j < EPL; ++j) mine = max(mine, key[j]);
    const uint32_t mx = wave_max(mine);
    if (mx == 0u) break;  // uniform: no open expert is left
    const int win = __builtin_ctzll(__ballot(mine == mx));
    bool left = lane == win;
#pragma unroll
    for (int j = 0; j < EPL; ++j) {
      const bool take = left && key[j] == mx;
      sel[j] = sel[j] || take;
      key[j] = take ? 0u : key[j];
      left = left && !take;
    }
    ++n_sel;
  }
  const uint64_t below = lane == 0 ? 0ull : (~0ull >> (64 - lane));
  int pos = 0;
#pragma unroll
  for (int j = 0; j < EPL; ++j) pos += __popcll(__ballot(sel[j]) & below);
#pragma unroll
  for (int j = 0; j < EPL; ++j) {
    if (sel[j]) {
      s_sel[wave][pos] = s[j];
      s_id[wave][pos] = lane * EPL + j;
      ++pos;
    }
  }
  __syncthreads();
  float sum = 0.0f;  // in ascending expert order
  for (int r = 0; r < n_sel; ++r) sum += s_sel[wave][r];
  sum += 1e-20f;
  if (active && lane < k) {
    const bool there = lane < n_sel;
    const float p = there ? s_sel[wave][lane] : 0.0f;
    weights[(size_t)t * k + lane] = (renormalize ? __fdiv_rn(p, sum) : p) * scale;
    ids[(size_t)t * k + lane] = there ? s_id[wave][lane] : -1;
  }
}

template <int EPL, int DT, bool SOFTMAX>
__global__ void __launch_bounds__(64 * WAVES)
route_topk_backward_kernel(const float* __restrict__ grad, const void* __restrict__ logits, size_t row_stride,
                           const int32_t* __restrict__ ids, int T, int E, int k, int renormalize, float scale,
                           void* __restrict__ out) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int t = blockIdx.x * WAVES + wave;
  if (t >= T) return;
  const size_t row = (size_t)t * row_stride;
  float x[EPL], s[EPL], slope[EPL], d[EPL];
#pragma unroll
  for (int j = 0; j < EPL; ++j) {
    const int e = lane * EPL + j;
    x[j] = e < E ? load_as_f32<DT>(logits, row + e) : -INFINITY;
    d[j] = 0.0f;
  }
  if constexpr (SOFTMAX) {
    float m = -INFINITY;
#pragma unroll
    for (int j = 0; j < EPL; ++j) m = fmaxf(m, x[j]);
    m = wave_max(m);
    float sum = 0.0f;
#pragma unroll
    for (int j = 0; j < EPL; ++j) {
      s[j] = x[j] > -INFINITY ? exp_below<float>(x[j], m) : 0.0f;
      sum += s[j];
    }
    sum = wave_sum(sum);
    const float inv = sum > 0.0f ? 1.0f / sum : 0.0f;
#pragma unroll
    for (int j = 0; j < EPL; ++j) s[j] *= inv;
  } else {
#pragma unroll
    for (int j = 0; j < EPL; ++j) {
      // both factors from exp(-|x|): 1 - s keeps its digits where s is near 1
      const float q = x[j] > -INFINITY ? expf(-fabsf(x[j])) : 0.0f;
      const float a = 1.0f / (1.0f + q), b = q * a;
      s[j] = x[j] >= 0.0f ? a : b;
      slope[j] = a * b;
    }
  }
  // Lane r < k: pick r, its score and weight gradient.
  const int id = lane < k ? ids[(size_t)t * k + lane] : -1;
  const bool there = id >= 0 && id < E;
  const float g = there ? grad[(size_t)t * k + lane] : 0.0f;
  float p = 0.0f;
  {
    const int at = there ? id / EPL : 0, sub = there ? id % EPL : 0;
#pragma unroll
    for (int j = 0; j < EPL; ++j) {
      const float o = __shfl(s[j], at);
      p = sub == j ? o : p;
    }
    p = there ? p : 0.0f;
  }
  float ds = scale * g;
  if (renormalize) {
    const float inv = 1.0f / (wave_sum(p) + 1e-20f);
    ds = scale * ((g - wave_sum(g * p) * inv) * inv);
    ds = there ? ds : 0.0f;
  }
  for (int r = 0; r < k; ++r) {
    const int e = __builtin_amdgcn_readlane(there ? id : -1, r) - lane * EPL;
    const float dr = __uint_as_float((uint32_t)__builtin_amdgcn_readlane((int)__float_as_uint(ds), r));
#pragma unroll
    for (int j = 0; j < EPL; ++j) d[j] += e == j ? dr : 0.0f;
  }
  const float mean = SOFTMAX ? wave_sum(ds * p) : 0.0f;
#pragma unroll
  for (int j = 0; j < EPL; ++j) {
    const int e = lane * EPL + j;
    if (e < E) store_f32_as<DT>(out, (size_t)t * E + e, SOFTMAX ? s[j] * (d[j] - mean) : d[j] * slope[j]);
  }
}

// f(integral_constant EPL, DT, SOFTMAX) for the launch's sizes.
template <class F>
hipError_t dispatch(int E, int dtype, int softmax, F&& f) {
  auto by_type = [&](auto epl) {
    auto by_score = [&](auto dt) {
      if (softmax) f(epl, dt, std::true_type{});
      else f(epl, dt, std::false_type{});
    };
    if (dtype == DT_F32) by_score(std::integral_constant<int, DT_F32>{});
    else if (dtype == DT_BF16) by_score(std::integral_constant<int, DT_BF16>{});
    else by_score(std::integral_constant<int, DT_F16>{});
  };
  if (E <= 64) by_type(std::integral_constant<int, 1>{});
  else if (E <= 128) by_type(std::integral_constant<int, 2>{});
  else if (E <= 256) by_type(std::integral_constant<int, 4>{});
  else if (E <= 512) by_type(std::integral_constant<int, 8>{});
  else by_type(std::integral_constant<int, 16>{});
  return hipGetLastError();
}

}  // namespace

hipError_t launch_route_topk(const void* logits, int dtype, size_t row_stride, const float* bias, int T, int E, int k,
                             int softmax, int n_group, int topk_group, int group_top, int renormalize, float scale,
                             float* weights, int32_t* ids, hipStream_t stream) {
  return dispatch(E, dtype, softmax, [&](auto epl, auto dt, auto sm) {
    constexpr int EPL = decltype(epl)::value;
    const int gs = E / n_group, lanes = gs / EPL;
    const bool whole = gs % EPL == 0 && lanes <= 16 && (lanes & (lanes - 1)) == 0;
    route_topk_kernel<decltype(epl)::value, decltype(dt)::value, decltype(sm)::value>
        <<<(T + WAVES - 1) / WAVES, 64 * WAVES, 0, stream>>>(logits, row_stride, bias, T, E, k, n_group,
                                                             whole ? lanes : 0, topk_group, group_top, renormalize,
                                                             scale, weights, ids);
  });
}

hipError_t launch_route_topk_backward(const float* grad, const void* logits, int dtype, size_t row_stride,
                                      const int32_t* ids, int T, int E, int k, int softmax, int renormalize,
                                      float scale, void* grad_logits, hipStream_t stream) {
  return dispatch(E, dtype, softmax, [&](auto epl, auto dt, auto sm) {
    route_topk_backward_kernel<decltype(epl)::value, decltype(dt)::value, decltype(sm)::value>
        <<<(T + WAVES - 1) / WAVES, 64 * WAVES, 0, stream>>>(grad, logits, row_stride, ids, T, E, k, renormalize,
                                                             scale, grad_logits);
  });
}

}  // namespace moe
