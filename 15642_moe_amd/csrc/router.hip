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
// The picks follow from comparisons of 32-bit values, so the 64-bit exponential, rounded
// once, is what makes them the same on every machine.
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

template <int DT>
__device__ __forceinline__ void store_4(void* base, size_t i, const float (&v)[4]) {  // aligned to the four
  if constexpr (DT == DT_F32) {
    *reinterpret_cast<float4*>(static_cast<float*>(base) + i) = make_float4(v[0], v[1], v[2], v[3]);
  } else {
    uint16_t h[4];
#pragma unroll
    for (int q = 0; q < 4; ++q) store_f32_as<DT>(h, q, v[q]);
    *reinterpret_cast<uint2*>(static_cast<uint16_t*>(base) + i) =
        make_uint2(h[0] | (uint32_t)h[1] << 16, h[2] | (uint32_t)h[3] << 16);
  }
}

// P consecutive elements, in loads of up to 16 bytes (the pointer aligned to them).
template <int DT, int P>
__device__ __forceinline__ void load_all(const void* base, size_t i, float (&x)[P]) {
  if constexpr (DT == DT_F32) {
#pragma unroll
    for (int j = 0; j < P; j += 4) {
      const float4 f = *reinterpret_cast<const float4*>(static_cast<const float*>(base) + i + j);
      x[j] = f.x; x[j + 1] = f.y; x[j + 2] = f.z; x[j + 3] = f.w;
    }
  } else {
#pragma unroll
    for (int j = 0; j < P; j += 4) {
      const uint2 u = *reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(base) + i + j);
      const uint32_t h[4] = {u.x & 0xFFFFu, u.x >> 16, u.y & 0xFFFFu, u.y >> 16};
#pragma unroll
      for (int q = 0; q < 4; ++q)
        x[j + q] = DT == DT_BF16 ? __uint_as_float(h[q] << 16) : (float)__builtin_bit_cast(_Float16, (uint16_t)h[q]);
    }
  }
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

// exp(x) to about 2^-52: x = n ln 2 + r with |r| <= ln(2) / 2 (ln 2 in two parts), and the
// series of exp(r) to r^13 / 13! (what is left is under 2^-57).
__device__ __forceinline__ double exp64(double x) {
  x = fmin(fmax(x, -1100.0), 1100.0);  // past both ends of the range
  const double n = rint(x * 0x1.71547652b82fep+0);
  double r = fma(n, -0x1.62e42fefa3800p-1, x);
  r = fma(n, -0x1.ef35793c76730p-45, r);
  double p = 1.0 / 6227020800.0;
  p = fma(p, r, 1.0 / 479001600.0);
  p = fma(p, r, 1.0 / 39916800.0);
  p = fma(p, r, 1.0 / 3628800.0);
  p = fma(p, r, 1.0 / 362880.0);
  p = fma(p, r, 1.0 / 40320.0);
  p = fma(p, r, 1.0 / 5040.0);
  p = fma(p, r, 1.0 / 720.0);
  p = fma(p, r, 1.0 / 120.0);
  p = fma(p, r, 1.0 / 24.0);
  p = fma(p, r, 1.0 / 6.0);
  p = fma(p, r, 0.5);
  p = fma(p, r, 1.0);
  p = fma(p, r, 1.0);
  return __builtin_amdgcn_ldexp(p, (int)n);
}

// exp(x - m) of a softmax; the maximum's own is 1, also where it is +inf.
__device__ __forceinline__ double exp64_below(float x, float m) { return x == m ? 1.0 : exp64((double)x - (double)m); }
__device__ __forceinline__ float exp32_below(float x, float m) { return x == m ? 1.0f : expf(x - m); }

// 1 / (1 + e), e = exp(-x) rounded once to 32 bits.
__device__ __forceinline__ float sigmoid(float x) { return __fdiv_rn(1.0f, 1.0f + (float)exp64(-(double)x)); }

struct RouteArgs {
  const void* logits;
  size_t row_stride;
  const float* bias;
  int T, E, k, n_group, lanes_per_group, topk_group, group_top, renormalize, vec;
  float scale;
  float* weights;
  int32_t* ids;
};
template <int EPL>
struct RouteLds {  // one wave's
  float v[64 * EPL];
  float sel[64];
  int id[64];
};
// Orders a wave's own LDS writes and reads (which the hardware keeps in order).
__device__ __forceinline__ void wave_fence() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

// Token t by one wave; lane l holds experts EPL*l .. +EPL.  Bound by the latency of k
// rounds of a wave-wide maximum: 256 experts in 8 groups, top 8, T = 1 in 4.3 us.
template <int EPL, int DT, bool SOFTMAX>
__device__ __forceinline__ void route_token(const RouteArgs& a, int t, RouteLds<EPL>& s) {
  const int lane = threadIdx.x & 63;
  const size_t row = (size_t)t * a.row_stride;
  float x[EPL], sc[EPL], v[EPL];
#pragma unroll
  for (int j = 0; j < EPL; ++j) {
    const int e = lane * EPL + j;
    x[j] = e < a.E ? load_as_f32<DT>(a.logits, row + e) : -INFINITY;
  }
  if constexpr (SOFTMAX) {
    float m = -INFINITY;
#pragma unroll
    for (int j = 0; j < EPL; ++j) m = fmaxf(m, x[j]);
    m = wave_max(m);
    double ex[EPL], sum = 0.0;
#pragma unroll
    for (int j = 0; j < EPL; ++j) {
      ex[j] = x[j] > -INFINITY ? exp64_below(x[j], m) : 0.0;
      sum += ex[j];
    }
    sum = wave_sum(sum);
    const double inv = sum > 0.0 ? 1.0 / sum : 0.0;
#pragma unroll
    for (int j = 0; j < EPL; ++j) sc[j] = (float)(ex[j] * inv);
  } else {
#pragma unroll
    for (int j = 0; j < EPL; ++j) sc[j] = sigmoid(x[j]);
  }
#pragma unroll
  for (int j = 0; j < EPL; ++j) {
    const int e = lane * EPL + j;
    v[j] = x[j] > -INFINITY ? (a.bias ? sc[j] + a.bias[e] : sc[j]) : -INFINITY;
    if (!(v[j] > -INFINITY)) v[j] = -INFINITY;
  }

  uint32_t key[EPL];
#pragma unroll
  for (int j = 0; j < EPL; ++j) key[j] = open_key(v[j]);
  if (a.n_group > 1) {
    const int gs = a.E / a.n_group;
    float m1 = -INFINITY, m2 = -INFINITY;
    auto score = [&] {  // a closed second place adds nothing
      return open_key((a.group_top == 2 && m2 > -INFINITY) ? m1 + m2 : m1);
    };
    auto add = [&](float y) {
      m2 = fmaxf(m2, fminf(m1, y));
      m1 = fmaxf(m1, y);
    };
    auto merge = [&](float o1, float o2) {
      m2 = fmaxf(fminf(m1, o1), fmaxf(m2, o2));
      m1 = fmaxf(m1, o1);
    };
    if (a.lanes_per_group > 0) {
      // A group is a power of two of whole lanes, at most a row's 16: its lanes merge
      // their two largest by DPP moves.
#pragma unroll
      for (int j = 0; j < EPL; ++j) add(v[j]);
      if (a.lanes_per_group > 1) merge(dpp<DPP_XOR1>(m1), dpp<DPP_XOR1>(m2));
      if (a.lanes_per_group > 2) merge(dpp<DPP_XOR2>(m1), dpp<DPP_XOR2>(m2));
      if (a.lanes_per_group > 4) merge(dpp<DPP_HALF_MIRROR>(m1), dpp<DPP_HALF_MIRROR>(m2));
      if (a.lanes_per_group > 8) merge(dpp<DPP_MIRROR>(m1), dpp<DPP_MIRROR>(m2));
      const uint32_t gkey = score();
      const int mine = lane / a.lanes_per_group;
      int rank = 0;
      for (int g = 0; g < a.n_group; ++g) {
        const uint32_t o = lane_of(gkey, g * a.lanes_per_group);
        rank += (o > gkey || (o == gkey && g < mine)) ? 1 : 0;
      }
      if (rank >= a.topk_group || mine >= a.n_group) {
#pragma unroll
        for (int j = 0; j < EPL; ++j) key[j] = 0u;
      }
    } else {
      // Lane g scores group g from LDS.
#pragma unroll
      for (int j = 0; j < EPL; ++j) s.v[lane * EPL + j] = v[j];
      wave_fence();
      if (lane < a.n_group)
        for (int i = 0; i < gs; ++i) add(s.v[lane * gs + i]);
      const uint32_t gkey = score();
      int rank = 0;
      for (int g = 0; g < a.n_group; ++g) {
        const uint32_t o = lane_of(gkey, g);
        rank += (o > gkey || (o == gkey && g < lane)) ? 1 : 0;
      }
      const uint64_t kept = __ballot(lane < a.n_group && rank < a.topk_group);
#pragma unroll
      for (int j = 0; j < EPL; ++j) {
        const int e = lane * EPL + j;
        if (e >= a.E || !((kept >> (e / gs)) & 1u)) key[j] = 0u;
      }
    }
  }

  bool sel[EPL];
#pragma unroll
  for (int j = 0; j < EPL; ++j) sel[j] = false;
  int n_sel = 0;
  for (int r = 0; r < a.k; ++r) {
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
      s.sel[pos] = sc[j];
      s.id[pos] = lane * EPL + j;
      ++pos;
    }
  }
  wave_fence();
  float sum = 0.0f;  // in ascending expert order
  for (int r = 0; r < n_sel; ++r) sum += s.sel[r];
  sum += 1e-20f;
  if (lane < a.k) {
    const bool there = lane < n_sel;
    const float p = there ? s.sel[lane] : 0.0f;
    a.weights[(size_t)t * a.k + lane] = (a.renormalize ? __fdiv_rn(p, sum) : p) * a.scale;
    a.ids[(size_t)t * a.k + lane] = there ? s.id[lane] : -1;
  }
}

template <int EPL, int DT, bool SOFTMAX>
__global__ void __launch_bounds__(64 * WAVES)
route_topk_kernel(RouteArgs a) {
  __shared__ RouteLds<EPL> s[WAVES];
  const int wave = threadIdx.x >> 6, t = blockIdx.x * WAVES + wave;
  if (t < a.T) route_token<EPL, DT, SOFTMAX>(a, t, s[wave]);
}

// ---------------------------------------------------------------------------
// Many tokens: four per wave, 16 lanes each, P experts a lane, the same scores and picks.
// One token per wave spends most of its instructions on wave-wide maxima of mostly idle
// lanes; here a lane sorts its experts once and a round of the selection is a row's
// maximum (four DPP moves for four tokens) and a pop of the winner's list.  Ties, which
// go to the lower expert, and groups that tie are told by counts and take a longer way.
// From T = 4096 on, where it takes less; us, one token a wave / four:
//   256 experts in 8 groups, sigmoid  T=2048 6.0 / 7.3, 4096 8.2 / 7.4, 16384 22.6 / 16.9
//   160 in 8, softmax, bf16           T=2048 6.7 / 8.7, 4096 9.3 / 9.0, 16384 25.8 / 16.8
//   64, softmax, bf16                 T=2048 3.5 / 4.0, 4096 4.4 / 4.1, 16384 10.4 / 7.0
// What bounds it is the vector unit: about 20 f64 instructions a score, 10 for the
// division, 20 a score for the selection; 17 MB of logits would take 3.4 us.
// ---------------------------------------------------------------------------
__device__ __forceinline__ void order(uint32_t& a, uint32_t& b) {  // a >= b
  const uint32_t hi = max(a, b), lo = min(a, b);
  a = hi;
  b = lo;
}
__device__ __forceinline__ void sort4(uint32_t* r) {
  order(r[0], r[1]); order(r[2], r[3]); order(r[0], r[2]); order(r[1], r[3]); order(r[1], r[2]);
}
__device__ __forceinline__ void sort8(uint32_t* r) {  // odd-even merge sort
  sort4(r);
  sort4(r + 4);
#pragma unroll
  for (int i = 0; i < 4; ++i) order(r[i], r[i + 4]);
  order(r[2], r[4]); order(r[3], r[5]);
  order(r[1], r[2]); order(r[3], r[4]); order(r[5], r[6]);
}
// Row-wide (16 lanes) reductions, the result in every lane of the row.
__device__ __forceinline__ uint32_t row_max(uint32_t x) {
  return dpp_max<DPP_MIRROR>(dpp_max<DPP_HALF_MIRROR>(dpp_max<DPP_XOR2>(dpp_max<DPP_XOR1>(x))));
}
__device__ __forceinline__ float row_max(float x) {
  x = fmaxf(x, dpp<DPP_XOR1>(x));
  x = fmaxf(x, dpp<DPP_XOR2>(x));
  x = fmaxf(x, dpp<DPP_HALF_MIRROR>(x));
  return fmaxf(x, dpp<DPP_MIRROR>(x));
}
template <class N>
__device__ __forceinline__ N row_sum(N x) {
  x += dpp<DPP_XOR1>(x);
  x += dpp<DPP_XOR2>(x);
  x += dpp<DPP_HALF_MIRROR>(x);
  return x + dpp<DPP_MIRROR>(x);
}
template <int N>
__device__ __forceinline__ int row_shr(int x) {  // lane i: lane i - N's, 0 below
  return __builtin_amdgcn_update_dpp(0, x, 0x110 + N, 0xF, 0xF, false);
}
template <int R>
__device__ __forceinline__ uint32_t row_ror(uint32_t x) {
  return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x120 + R, 0xF, 0xF, false);
}
// Lanes of the row with a larger key, and with TIES those with an equal one below this.
template <bool TIES, int R = 1>
__device__ __forceinline__ int lanes_above(uint32_t key, uint32_t sub) {
  if constexpr (R == 16) {
    return 0;
  } else {
    // Both moves before any branch: a lane that is switched off has nothing to move.
    const uint32_t o = row_ror<R>(key), o_sub = TIES ? row_ror<R>(sub) : 0u;
    const bool above = (o > key) | (TIES & (o == key) & (o_sub < sub));
    return (above ? 1 : 0) + lanes_above<TIES, R + 1>(key, sub);
  }
}
// Sum of the lanes below in the row.
__device__ __forceinline__ int row_below(int x) {
  int s = x;
  s += row_shr<1>(s);
  s += row_shr<2>(s);
  s += row_shr<4>(s);
  s += row_shr<8>(s);
  return s - x;
}

constexpr int ROWS_MAX_K = 8, ROWS_MIN_T = 4096;
template <int P, int DT, bool SOFTMAX>
__global__ void __launch_bounds__(64 * WAVES)
route_rows_kernel(RouteArgs a) {
  constexpr int LIST = P < ROWS_MAX_K ? P : ROWS_MAX_K;
  __shared__ int s_id[WAVES][4][ROWS_MAX_K];
  __shared__ float s_sel[WAVES][4][ROWS_MAX_K];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, row = lane >> 4, sub = lane & 15;
  const int t0 = (blockIdx.x * WAVES + wave) * 4;
  if (t0 >= a.T) return;  // uniform
  const int t = min(t0 + row, a.T - 1), per = (a.E + 15) >> 4, e0 = sub * per;
  const size_t at = (size_t)t * a.row_stride;
  float x[P], v[P];
  if (a.vec) {
    load_all<DT, P>(a.logits, at + e0, x);
  } else {
#pragma unroll
    for (int j = 0; j < P; ++j) x[j] = j < per && e0 + j < a.E ? load_as_f32<DT>(a.logits, at + e0 + j) : -INFINITY;
  }
  float m = -INFINITY;
  double inv = 0.0;
  if constexpr (SOFTMAX) {
#pragma unroll
    for (int j = 0; j < P; ++j) m = fmaxf(m, x[j]);
    m = row_max(m);
    double ex[P], sum = 0.0;
#pragma unroll
    for (int j = 0; j < P; ++j) {
      ex[j] = x[j] > -INFINITY ? exp64_below(x[j], m) : 0.0;
      sum += ex[j];
    }
    sum = row_sum(sum);
    inv = sum > 0.0 ? 1.0 / sum : 0.0;
#pragma unroll
    for (int j = 0; j < P; ++j) v[j] = (float)(ex[j] * inv);
  } else {
#pragma unroll
    for (int j = 0; j < P; ++j) v[j] = sigmoid(x[j]);
  }
  if (a.bias) {
    if (a.vec) {
      float b[P];
      load_all<DT_F32, P>(a.bias, e0, b);
#pragma unroll
      for (int j = 0; j < P; ++j) v[j] += b[j];
    } else {
#pragma unroll
      for (int j = 0; j < P; ++j)
        if (j < per && e0 + j < a.E) v[j] += a.bias[e0 + j];
    }
  }
  uint32_t key[P];
#pragma unroll
  for (int j = 0; j < P; ++j) key[j] = x[j] > -INFINITY ? open_key(v[j]) : 0u;
  if (a.n_group > 1) {
    const int lpg = a.lanes_per_group;
    float m1 = -INFINITY, m2 = -INFINITY;
#pragma unroll
    for (int j = 0; j < P; ++j) {
      const float y = key[j] ? v[j] : -INFINITY;
      m2 = fmaxf(m2, fminf(m1, y));
      m1 = fmaxf(m1, y);
    }
    auto merge = [&](float o1, float o2) {
      m2 = fmaxf(fminf(m1, o1), fmaxf(m2, o2));
      m1 = fmaxf(m1, o1);
    };
    if (lpg > 1) merge(dpp<DPP_XOR1>(m1), dpp<DPP_XOR1>(m2));
    if (lpg > 2) merge(dpp<DPP_XOR2>(m1), dpp<DPP_XOR2>(m2));
    if (lpg > 4) merge(dpp<DPP_HALF_MIRROR>(m1), dpp<DPP_HALF_MIRROR>(m2));
    const uint32_t score = open_key((a.group_top == 2 && m2 > -INFINITY) ? m1 + m2 : m1);
    const int most = a.topk_group * lpg;
    bool kept = lanes_above<false>(score, sub) < most;
    // Groups that tie for the last place are all kept so far.
    if (__any(row_sum(kept && score ? 1 : 0) > most)) kept = lanes_above<true>(score, sub) < most;
#pragma unroll
    for (int j = 0; j < P; ++j) key[j] = kept ? key[j] : 0u;
  }
  // The k-th largest: every lane's largest in order, then k times the row's largest head.
  uint32_t r[P < 8 ? 8 : P];
#pragma unroll
  for (int j = 0; j < P; ++j) r[j] = key[j];
  if constexpr (P == 4) {
    sort4(r);
  } else {
    sort8(r);
  }
  if constexpr (P == 16) {
    sort8(r + 8);
#pragma unroll
    for (int i = 0; i < 8; ++i) r[i] = max(r[i], r[15 - i]);  // the 8 largest, a bitonic sequence
#pragma unroll
    for (int d = 4; d > 0; d >>= 1)
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (!(i & d)) order(r[i], r[i + d]);
  }
  uint32_t kth = 0;
#pragma unroll
  for (int i = 0; i < ROWS_MAX_K; ++i) {
    if (i < a.k) {
      kth = row_max(r[0]);
      const uint32_t heads = (uint32_t)(__ballot(r[0] == kth) >> (row * 16)) & 0xFFFFu;
      const bool pop = (heads & -heads) == 1u << sub;  // the first of the lanes that have it
      // The empty asm keeps the list in its registers: the compiler would turn the moves
      // into a search for the r[pops so far], 16 comparisons a round.
#pragma unroll
      for (int j = 0; j < LIST; ++j)
        if (j < ROWS_MAX_K - i) {  // as far as the rounds to come reach
          r[j] = pop ? (j + 1 < LIST ? r[j + 1] : 0u) : r[j];
          __asm__("" : "+v"(r[j]));
        }
    }
  }
  uint32_t mask = 0;  // the picks
#pragma unroll
  for (int j = 0; j < P; ++j) mask |= (key[j] >= kth && key[j] ? 1u : 0u) << j;
  int n = row_sum((int)__popc(mask));
  if (__any(n > a.k)) {  // equals of the k-th are too many: the lower ones stay
    uint32_t equal = 0;
#pragma unroll
    for (int j = 0; j < P; ++j) equal |= (key[j] == kth && key[j] ? 1u : 0u) << j;
    const int n_equal = row_sum((int)__popc(equal)), room = a.k - (n - n_equal);
    int left = room - row_below((int)__popc(equal));
    mask &= ~equal;
    for (; equal && left > 0; equal &= equal - 1, --left) mask |= equal & -equal;
    n = row_sum((int)__popc(mask));
  }
  int pos = row_below((int)__popc(mask));
  for (; mask; mask &= mask - 1) s_id[wave][row][pos++] = e0 + __builtin_ctz(mask);
  wave_fence();
  const int id = sub < n ? s_id[wave][row][sub] : -1;  // n <= k <= 8
  float p = 0.0f;
  if (id >= 0) {
    const float xi = load_as_f32<DT>(a.logits, at + id);
    if constexpr (SOFTMAX) p = (float)(exp64_below(xi, m) * inv);
    else p = sigmoid(xi);
  }
  if (sub < ROWS_MAX_K) s_sel[wave][row][sub] = p;
  wave_fence();
  float total = 0.0f;  // in ascending expert order
#pragma unroll
  for (int i = 0; i < ROWS_MAX_K; ++i) total += s_sel[wave][row][i];
  total += 1e-20f;
  if (t0 + row < a.T && sub < a.k) {
    a.weights[(size_t)t * a.k + sub] = (a.renormalize ? __fdiv_rn(p, total) : p) * a.scale;
    a.ids[(size_t)t * a.k + sub] = id;
  }
}

// ---------------------------------------------------------------------------
// The gradient: L = 16 or 64 lanes a token, a lane the experts 4 (i L + l) .. +4 of each
// piece i, so that loads and stores are whole lines.  The picks' gradients, a lane each,
// go to the token's row in LDS; with sigmoid they are the result (only the picks' logits
// are read), with softmax each expert's share of the normaliser is added to them.
// ---------------------------------------------------------------------------
template <int L, class N>
__device__ __forceinline__ N lanes_sum(N x) {
  if constexpr (L == 16) return row_sum(x);
  else return wave_sum(x);
}
template <int L, int P, int DT, bool SOFTMAX>
__global__ void __launch_bounds__(64 * WAVES)
route_topk_backward_kernel(const float* __restrict__ grad, const void* __restrict__ logits, size_t row_stride,
                           const int32_t* __restrict__ ids, int T, int E, int k, int renormalize, float scale,
                           int vec, void* __restrict__ out) {
  constexpr int TOKENS = 64 / L;  // a wave's
  __shared__ __align__(16) float s_d[WAVES][TOKENS][L * P];
  __shared__ int2 s_pick[WAVES][TOKENS][L];  // id, gradient
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, row = lane / L, sub = lane % L;
  const int t0 = (blockIdx.x * WAVES + wave) * TOKENS;
  if (t0 >= T) return;  // uniform
  const int t = min(t0 + row, T - 1);
  const size_t at = (size_t)t * row_stride;
  float* d = s_d[wave][row];
  int2* picks = s_pick[wave][row];
  // Lane r < k: pick r.
  int id = sub < k ? ids[(size_t)t * k + sub] : -1;
  if (id >= E) id = -1;
  const float g = id >= 0 ? grad[(size_t)t * k + sub] : 0.0f;
  float s[P], m = -INFINITY, inv = 0.0f;
  if constexpr (SOFTMAX) {
#pragma unroll
    for (int i = 0; i < P / 4; ++i) {
      const int e = 4 * (i * L + sub);
      float x[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
      if (vec) {
        if (e < E) load_all<DT, 4>(logits, at + e, x);
      } else {
#pragma unroll
        for (int q = 0; q < 4; ++q)
          if (e + q < E) x[q] = load_as_f32<DT>(logits, at + e + q);
      }
#pragma unroll
      for (int q = 0; q < 4; ++q) s[i * 4 + q] = x[q];
    }
  }
  const float xp = id >= 0 ? load_as_f32<DT>(logits, at + id) : -INFINITY;
#pragma unroll
  for (int i = 0; i < P / 4; ++i)
    if (i * 4 * L < E) *reinterpret_cast<float4*>(d + 4 * (i * L + sub)) = make_float4(0.f, 0.f, 0.f, 0.f);
  float p, slope = 0.0f;
  if constexpr (SOFTMAX) {
#pragma unroll
    for (int j = 0; j < P; ++j) m = fmaxf(m, s[j]);
    if constexpr (L == 16) m = row_max(m);
    else m = wave_max(m);
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < P / 4; ++i) {
      if (i * 4 * L < E) {
#pragma unroll
        for (int j = 4 * i; j < 4 * i + 4; ++j) {
          s[j] = s[j] > -INFINITY ? exp32_below(s[j], m) : 0.0f;
          sum += s[j];
        }
      }
    }
    sum = lanes_sum<L>(sum);
    inv = sum > 0.0f ? 1.0f / sum : 0.0f;
    p = xp > -INFINITY ? exp32_below(xp, m) * inv : 0.0f;
  } else {
    // both factors from exp(-|x|): 1 - s keeps its digits where s is near 1
    const float q = xp > -INFINITY ? expf(-fabsf(xp)) : 0.0f;
    const float a = 1.0f / (1.0f + q), b = q * a;
    p = xp >= 0.0f ? a : b;
    slope = a * b;
  }
  float ds = scale * g;
  if (renormalize) {
    const float inv_p = 1.0f / (lanes_sum<L>(p) + 1e-20f);
    const float part = lanes_sum<L>(g * p) * inv_p;  // by all lanes: before the choice
    ds = id >= 0 ? scale * ((g - part) * inv_p) : 0.0f;
  }
  const float mean = SOFTMAX ? lanes_sum<L>(ds * p) : 0.0f;
  const float mine = SOFTMAX ? ds : ds * slope;
  picks[sub] = make_int2(id, __float_as_int(mine));
  wave_fence();
  // A pick that stands in several slots: each of them writes the sum over all, in their
  // order.  (Slots up to the next multiple of 8 are there, and empty.)
  float all = 0.0f;
  for (int r0 = 0; r0 < k; r0 += 8) {
#pragma unroll
    for (int r = 0; r < 8; ++r) {
      const int2 o = picks[r0 + r];
      all += o.x == id ? __int_as_float(o.y) : 0.0f;
    }
  }
  if (id >= 0) d[id] = all;
  wave_fence();
  if (t0 + row >= T) return;
#pragma unroll
  for (int i = 0; i < P / 4; ++i) {
    const int e = 4 * (i * L + sub);
    if (e >= E) break;
    const float4 u = *reinterpret_cast<const float4*>(d + e);
    float y[4] = {u.x, u.y, u.z, u.w};
    if constexpr (SOFTMAX) {
#pragma unroll
      for (int q = 0; q < 4; ++q) y[q] = s[i * 4 + q] * inv * (y[q] - mean);
    }
    if (vec) {
      store_4<DT>(out, (size_t)t * E + e, y);
    } else {
#pragma unroll
      for (int q = 0; q < 4; ++q)
        if (e + q < E) store_f32_as<DT>(out, (size_t)t * E + e + q, y[q]);
    }
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

// Lanes of `per` experts that make up a group, if they are a power of two of whole
// lanes, at most `most`; else 0.
static int whole_lanes(int group, int per, int most) {
  const int lanes = group / per;
  return group % per == 0 && lanes <= most && (lanes & (lanes - 1)) == 0 ? lanes : 0;
}

hipError_t launch_route_topk(const void* logits, int dtype, size_t row_stride, const float* bias, int T, int E, int k,
                             int softmax, int n_group, int topk_group, int group_top, int renormalize, float scale,
                             float* weights, int32_t* ids, hipStream_t stream) {
  RouteArgs a = {logits, row_stride, bias, T, E, k, n_group, 0, topk_group, group_top, renormalize, 0, scale, weights, ids};
  const int per = (E + 15) / 16, rows_lanes = n_group > 1 ? whole_lanes(E / n_group, per, 8) : 1;
  if (T >= ROWS_MIN_T && E <= 256 && k <= ROWS_MAX_K && rows_lanes > 0) {
    a.lanes_per_group = rows_lanes;
    const size_t size = dtype == DT_F32 ? 4 : 2;  // loads of 4 elements
    a.vec = (E == 64 || E == 128 || E == 256) && row_stride % 4 == 0 && (uintptr_t)logits % (4 * size) == 0 &&
            (uintptr_t)bias % 16 == 0;
    return dispatch(E, dtype, softmax, [&](auto epl, auto dt, auto sm) {
      constexpr int EPL = decltype(epl)::value;
      if constexpr (EPL <= 4)
        route_rows_kernel<4 * EPL, decltype(dt)::value, decltype(sm)::value>
            <<<(T + 4 * WAVES - 1) / (4 * WAVES), 64 * WAVES, 0, stream>>>(a);
    });
  }
  return dispatch(E, dtype, softmax, [&](auto epl, auto dt, auto sm) {
    constexpr int EPL = decltype(epl)::value;
    a.lanes_per_group = whole_lanes(E / n_group, EPL, 16);
    route_topk_kernel<EPL, decltype(dt)::value, decltype(sm)::value>
        <<<(T + WAVES - 1) / WAVES, 64 * WAVES, 0, stream>>>(a);
  });
}

hipError_t launch_route_topk_backward(const float* grad, const void* logits, int dtype, size_t row_stride,
                                      const int32_t* ids, int T, int E, int k, int softmax, int renormalize,
                                      float scale, void* grad_logits, hipStream_t stream) {
  const size_t size = dtype == DT_F32 ? 4 : 2;  // loads and stores of 4 elements
  const int vec = E % 4 == 0 && row_stride % 4 == 0 && (uintptr_t)logits % (4 * size) == 0;
  // 16 lanes a token where there are tokens enough; us, 64 lanes / 16:
  //   160 experts, softmax, bf16  T=2048 3.2 / 4.1, 4096 4.0 / 4.3, 8192 5.5 / 4.7, 16384 8.8 / 6.4
  //   100, softmax, f32           T=2048 3.3 / 3.5, 4096 4.2 / 3.7, 16384 9.5 / 5.5
  //   60, softmax, bf16           T=1024 3.1 / 3.0, 4096 4.2 / 3.1, 16384 9.3 / 4.1
  //   256, sigmoid, f32           T=2048 2.8 / 3.0, 16384 7.0 / 7.0: always 64
  // What bounds it at T = 16384 is the memory's latency and 16 exponentials a lane; 160
  // experts' 10.5 MB in and out would take 2.0 us.
  const bool rows = E <= 256 && k <= 16 && T >= 32 * E;
  return dispatch(E, dtype, softmax, [&](auto epl, auto dt, auto sm) {
    constexpr int EPL = decltype(epl)::value, DT = decltype(dt)::value;
    constexpr bool SOFTMAX = decltype(sm)::value;
    auto launch = [&](auto kernel, int tokens) {
      kernel<<<(T + tokens - 1) / tokens, 64 * WAVES, 0, stream>>>(grad, logits, row_stride, ids, T, E, k, renormalize,
                                                                   scale, vec, grad_logits);
    };
    if constexpr (EPL <= 4 && SOFTMAX) {
      if (rows) return launch(route_topk_backward_kernel<16, 4 * EPL, DT, SOFTMAX>, 4 * WAVES);
    }
    launch(route_topk_backward_kernel<64, EPL < 4 ? 4 : EPL, DT, SOFTMAX>, WAVES);
  });
}

}  // namespace moe
