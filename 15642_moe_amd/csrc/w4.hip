// 4-bit weights: OCP MXFP4 (e2m1 codes, one e8m0 scale per 32 elements of K) on
// block-scaled e4m3 activations (one fp32 scale per 128 elements of K).
//
//   y[t, n] = sum_kb xs[kb, t] * sum_{k in block kb} x[t, k] * 2^(sc[n, k/32] - 127) * e2m1(code[n, k])
//
// The inner sum of a 128-block is one v_mfma_scale_f32_16x16x128_f8f6f4 with
// the weights as the fp4 A operand, whose e8m0 scales the instruction applies,
// and the activations as the e4m3 B operand: no dequantisation, and one
// fp32 multiply-add per output and K-block for the activation scale.
//
// What bounds the products at few tokens is the weights' stream, 4.25 bits
// each: half of the FP8 layer's bytes.
#include "common.h"
#include "launch.h"
#include "w4.h"

#include <type_traits>

namespace moe {
namespace {

typedef unsigned u32x4 __attribute__((ext_vector_type(4)));

// Workgroups of a launch whose kernel loops over what is left (a launch's
// threads have to stay below 2^32).
constexpr size_t MAX_GRID = (size_t)1 << 20;

// ---------------------------------------------------------------------------
// Layout.  A thread per 16 bytes of codes (and, of them, the first of a
// K-block per scale byte).
// ---------------------------------------------------------------------------
__global__ void __launch_bounds__(256)
pack_w4_kernel(uint8_t* __restrict__ codes, uint8_t* __restrict__ scales, uint8_t* __restrict__ packed, int N, int K,
               size_t units, int unpack) {
  const size_t u = (size_t)blockIdx.x * 256 + threadIdx.x;  // (matrix and 16-row tile, chunk, K-block, lane)
  if (u >= units) return;
  const int lane = u & 63, b = (u >> 6) & 3;
  const int KC = w4_chunks(K), NT = w4_tiles(N);
  const size_t q = u >> 8;  // packed chunk
  const int c = (int)(q % KC), tile = (int)(q / KC % NT);
  const size_t m = q / KC / NT;
  const int row = tile * 16 + (lane & 15), g = lane >> 4, kb = c * W4_CHUNK_BLOCKS + b;
  const bool there = row < N && kb * BLK < K;
  uint8_t* pc = packed + q * W4_CHUNK_BYTES + b * W4_BLOCK_BYTES + lane * 16;
  uint8_t* ps = packed + q * W4_CHUNK_BYTES + W4_CHUNK_BLOCKS * W4_BLOCK_BYTES + lane * 4 + b;
  const size_t src = (m * N + (there ? row : 0)) * (size_t)(K / 2) + (size_t)(there ? kb : 0) * (BLK / 2) + g * 16;
  const size_t ssrc = (m * N + (there ? row : 0)) * (size_t)(K / 32) + (size_t)(there ? kb : 0) * (BLK / 32) + g;
  if (unpack) {
    if (!there) return;
    *reinterpret_cast<uint4*>(codes + src) = *reinterpret_cast<const uint4*>(pc);
    scales[ssrc] = *ps;
  } else {
    // Padding rows and K-blocks: zero codes at scale 1.
    *reinterpret_cast<uint4*>(pc) = there ? *reinterpret_cast<const uint4*>(codes + src) : make_uint4(0, 0, 0, 0);
    *ps = there ? scales[ssrc] : (uint8_t)127;
  }
}

template <int DT>
__device__ __forceinline__ void load8(const void* base, size_t i, float (&f)[8]) {
  if constexpr (DT == DT_F32) {
    const float4 a = *reinterpret_cast<const float4*>(static_cast<const float*>(base) + i);
    const float4 b = *reinterpret_cast<const float4*>(static_cast<const float*>(base) + i + 4);
    f[0] = a.x; f[1] = a.y; f[2] = a.z; f[3] = a.w;
    f[4] = b.x; f[5] = b.y; f[6] = b.z; f[7] = b.w;
  } else {
    const u32x4 u = *reinterpret_cast<const u32x4*>(static_cast<const uint16_t*>(base) + i);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if constexpr (DT == DT_BF16) {
        f[2 * j] = __builtin_bit_cast(float, u[j] << 16);
        f[2 * j + 1] = __builtin_bit_cast(float, u[j] & 0xFFFF0000u);
      } else {
        f[2 * j] = (float)__builtin_bit_cast(_Float16, (uint16_t)u[j]);
        f[2 * j + 1] = (float)__builtin_bit_cast(_Float16, (uint16_t)(u[j] >> 16));
      }
    }
  }
}

// ---------------------------------------------------------------------------
// MXFP4 of a matrix, once per weight: the shared exponent of 32 elements is that of their
// largest magnitude less 2 (the OCP rule: it lands in [4, 8), of which e2m1
// reaches 6), codes rounded to nearest, ties to even, saturating.  A group with
// an infinity or NaN gets the NaN scale.  Four threads a group, 8 elements each, converted
// by v_cvt_scalef32_pk_fp4_f32.  Bound by the copy: 235 M bf16 elements in 109 us, 5.4 TB/s
// (174 with the codes counted from seven comparisons).
// ---------------------------------------------------------------------------
template <int DT>
__global__ void __launch_bounds__(256)
quantize_w4_kernel(const void* __restrict__ w, size_t groups, uint8_t* __restrict__ codes,
                   uint8_t* __restrict__ scales) {
  const size_t u = (size_t)blockIdx.x * 256 + threadIdx.x;
  const size_t grp = u >> 2;
  const bool active = grp < groups;
  float f[8];
  load8<DT>(w, (active ? u : 0) * 8, f);
  uint32_t m = 0;
#pragma unroll
  for (int j = 0; j < 8; ++j) m = max(m, __float_as_uint(f[j]) & 0x7FFFFFFFu);  // NaN above inf
  m = max(m, (uint32_t)__shfl_xor((int)m, 1));
  m = max(m, (uint32_t)__shfl_xor((int)m, 2));
  const bool bad = m >= 0x7F800000u;
  // e8m0 = (exponent field of the maximum) - 2, at least 0: a maximum below
  // 2^-125 keeps the smallest scale, 2^-127.
  const int ex = max((int)(m >> 23) - 2, 0);
  const float up = __uint_as_float((uint32_t)(254 - ex) << 23);  // 2^(127 - ex), exact to multiply by
  uint32_t packed = 0;  // at scale 1: two codes a byte
  packed = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(packed, f[0] * up, f[1] * up, 1.0f, 0);
  packed = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(packed, f[2] * up, f[3] * up, 1.0f, 1);
  packed = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(packed, f[4] * up, f[5] * up, 1.0f, 2);
  packed = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(packed, f[6] * up, f[7] * up, 1.0f, 3);
  if (!active) return;
  reinterpret_cast<uint32_t*>(codes)[u] = bad ? 0u : packed;
  if ((u & 3) == 0) scales[grp] = bad ? (uint8_t)255 : (uint8_t)ex;
}

// ---------------------------------------------------------------------------
// Activations: per (row, 128 columns) scale = max(amax / 448, 1e-8), code =
// e4m3(clamp(x / scale, +-448)), the rule of the producer and of the experts'
// own requantisation.  16 lanes a block, 8 columns each.  Bound by the copy: bf16, T = 8192,
// K = 7168 in 32 us, 5.5 TB/s (the first form, which divided and took a block at a time, 46).
// ---------------------------------------------------------------------------
// x / s correctly rounded wherever its e4m3 code can tell: from y = RN(1 / s) two
// steps of remainder and correction (Markstein's: the second starts from a quotient
// within an ulp), five operations where the IEEE division takes about ten.  x's sign is
// put back (the correction turns -0 into +0).  |x| is at most the block's maximum, so the
// quotient is at most 448 and an ulp or two, which e4m3 rounds to 448: no clamp.
// s is the scale clamped to FLT_MAX: beside an infinite scale (y = 0) finite elements
// become 0; infinities and NaN become NaN.
__device__ __forceinline__ float quot(float x, float s, float y) {
  const float q0 = x * y;
  const float q1 = __builtin_fmaf(__builtin_fmaf(-q0, s, x), y, q0);
  return __builtin_copysignf(__builtin_fmaf(__builtin_fmaf(-q1, s, x), y, q1), x);
}
__device__ __forceinline__ uint32_t quot4_e4m3(float a, float b, float c, float d, float s, float y) {
  return cvt4_e4m3(quot(a, s, y), quot(b, s, y), quot(c, s, y), quot(d, s, y));
}
// Scale of a block with the largest magnitude m, and what quot takes of it.
__device__ __forceinline__ float block_scale(float m, float& s, float& y) {
  const float sc = fmaxf(m / E4M3_MAX, 1.0e-8f);
  s = fminf(sc, __FLT_MAX__);
  y = 1.0f / sc;
  return sc;
}

__device__ __forceinline__ uint2 quant8(const float (&f)[8], float& sc) {
  float m = 0.0f;
#pragma unroll
  for (int j = 0; j < 8; ++j) m = fmaxf(m, fabsf(f[j]));
#pragma unroll
  for (int o = 1; o < 16; o <<= 1) m = fmaxf(m, __shfl_xor(m, o));
  float s, y;
  sc = block_scale(m, s, y);
  return make_uint2(quot4_e4m3(f[0], f[1], f[2], f[3], s, y), quot4_e4m3(f[4], f[5], f[6], f[7], s, y));
}

// A workgroup takes 16 rows x G blocks: a row's G blocks are read at once, and a block's
// 16 scales are one line of [K / 128, T].
template <int DT, int G>
__global__ void __launch_bounds__(256)
quant_act_kernel(const void* __restrict__ x, size_t row_stride, int T, int KB, uint8_t* __restrict__ codes,
                 float* __restrict__ scale) {
  const int t = blockIdx.x * 16 + (threadIdx.x >> 4), sub = threadIdx.x & 15, kb0 = blockIdx.y * G;
  const size_t row = (size_t)min(t, T - 1) * row_stride;
  float f[G][8];
#pragma unroll
  for (int i = 0; i < G; ++i) load8<DT>(x, row + (size_t)min(kb0 + i, KB - 1) * BLK + sub * 8, f[i]);
#pragma unroll
  for (int i = 0; i < G; ++i) {
    float sc;
    const uint2 o = quant8(f[i], sc);
    if (t < T && kb0 + i < KB) {
      *reinterpret_cast<uint2*>(codes + ((size_t)t * KB + kb0 + i) * BLK + sub * 8) = o;
      if (sub == 0) scale[(size_t)(kb0 + i) * T + t] = sc;
    }
  }
}

// The same for the experts' SwiGLU output: Cf [R, I] -> Cq [R, I], Cs [R, I / 128].
__global__ void __launch_bounds__(256)
requant_kernel(const float* __restrict__ Cf, const int32_t* __restrict__ n_routes, int IB, uint8_t* __restrict__ Cq,
               float* __restrict__ Cs) {
  const size_t n = (size_t)*n_routes * IB;
  const int sub = threadIdx.x & 15;
  for (size_t u0 = (size_t)blockIdx.x * 16; u0 < n; u0 += (size_t)gridDim.x * 16) {
    const size_t u = u0 + (threadIdx.x >> 4);
    const bool active = u < n;
    float f[8], sc;
    load8<DT_F32>(Cf, (active ? u : 0) * BLK + sub * 8, f);
    const uint2 o = quant8(f, sc);
    if (active) {
      *reinterpret_cast<uint2*>(Cq + u * BLK + sub * 8) = o;
      if (sub == 0) Cs[u] = sc;
    }
  }
}

// ---------------------------------------------------------------------------
// The products.  A wave multiplies NT 16-row weight tiles with FR fragments of
// 16 activation rows over its share of the chunks of 512 K elements; the
// waves of a workgroup split the chunks, and their sums are added in K order
// through LDS: at few rows the weights are what counts, and all of a workgroup's are in
// flight at once.  N = 4096, K = 7168 (15.6 MB): 3.9 us at T = 1, 4.0 TB/s with the
// launch; 6.7 at T = 16; 11.4 at T = 64.
// ---------------------------------------------------------------------------
template <int B>
__device__ __forceinline__ v4f mfma_w4(const u32x4& a, const v8i& x, int scale, const v4f& c) {
  v8i aw{};
  aw[0] = (int)a[0]; aw[1] = (int)a[1]; aw[2] = (int)a[2]; aw[3] = (int)a[3];
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(aw, x, c, 4, 0, B, scale, 0, 127);
}

template <int N, int I0 = 0, class F>
__device__ __forceinline__ void static_for(F&& f) {
  if constexpr (I0 < N) {
    f(std::integral_constant<int, I0>{});
    static_for<N, I0 + 1>(f);
  }
}

template <int NT, int FR>
struct Stream {
  const uint8_t* w[NT];   // packed tiles, this lane's 16 bytes of the first K-block
  const uint8_t* x[FR];   // this lane's activation row, at its 16 bytes of the first K-block
  const float* xs[FR];    // that row's scale of the first K-block
  size_t xs_stride;       // from one K-block's scale to the next
  u32x4 a[NT][4];
  int sc[NT];
  v4f acc[NT][FR];

  __device__ __forceinline__ void load(int c) {
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const uint8_t* p = w[n] + (size_t)c * W4_CHUNK_BYTES;
#pragma unroll
      for (int b = 0; b < 4; ++b)
        a[n][b] = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(p + b * W4_BLOCK_BYTES));
      sc[n] = __builtin_nontemporal_load(
          reinterpret_cast<const int*>(p + W4_CHUNK_BLOCKS * W4_BLOCK_BYTES - 12 * (threadIdx.x & 63)));
    }
  }
  // Chunks c0 .. c1 - 1 of KB K-blocks in all.
  __device__ __forceinline__ void run(int c0, int c1, int KB) {
    const v4f zero4 = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int f = 0; f < FR; ++f) acc[n][f] = zero4;
    if (c0 >= c1) return;
    load(c0);
    for (int c = c0; c < c1; ++c) {
      u32x4 ca[NT][4];
      int csc[NT];
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        csc[n] = sc[n];
#pragma unroll
        for (int b = 0; b < 4; ++b) ca[n][b] = a[n][b];
      }
      if constexpr (FR == 1) {
        // This chunk's activations, then the next one's weights: loads return in order,
        // and the wait for the former leaves the latter in flight.
        u32x4 lo[4], hi[4];
        float s[4];
#pragma unroll
        for (int b = 0; b < 4; ++b) fragment(min(c * W4_CHUNK_BLOCKS + b, KB - 1), 0, lo[b], hi[b], s[b]);
        if (c + 1 < c1) load(c + 1);
        static_for<4>([&](auto bc) __attribute__((always_inline)) {
          constexpr int b = decltype(bc)::value;
          if (c * W4_CHUNK_BLOCKS + b < KB) multiply<b>(0, ca, csc, lo[b], hi[b], s[b]);
        });
      } else {
        // By K-blocks: the registers of a chunk's fragments would cost half of the waves.
        if (c + 1 < c1) load(c + 1);
        static_for<4>([&](auto bc) __attribute__((always_inline)) {
          constexpr int b = decltype(bc)::value;
          const int kb = c * W4_CHUNK_BLOCKS + b;
          if (kb < KB) {
#pragma unroll
            for (int f = 0; f < FR; ++f) {
              u32x4 lo, hi;
              float s;
              fragment(kb, f, lo, hi, s);
              multiply<b>(f, ca, csc, lo, hi, s);
            }
          }
        });
      }
    }
  }
  __device__ __forceinline__ void fragment(int kb, int f, u32x4& lo, u32x4& hi, float& s) const {
    lo = *reinterpret_cast<const u32x4*>(x[f] + (size_t)kb * BLK);
    hi = *reinterpret_cast<const u32x4*>(x[f] + (size_t)kb * BLK + 64);
    s = xs[f][(size_t)kb * xs_stride];
  }
  template <int B>
  __device__ __forceinline__ void multiply(int f, const u32x4 (&ca)[NT][4], const int (&csc)[NT], const u32x4& lo,
                                           const u32x4& hi, float s) {
    const v4f zero4 = {0.f, 0.f, 0.f, 0.f};
    const v8i xb = __builtin_bit_cast(v8i, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
#pragma unroll
    for (int n = 0; n < NT; ++n) acc[n][f] += mfma_w4<B>(ca[n][B], xb, csc[n], zero4) * s;
  }
  // The workgroup's sums, entry (n, f) in the registers of the wave that owns
  // it: `own(entry)` is called for the entries of this wave, after the waves'
  // parts have been added in K order.  Entries come as groups of G tiles (a
  // gate and an up tile for GEMM1): group p holds tiles p, p + NT / G, ...
  template <int G, class F>
  __device__ __forceinline__ void reduce(v4f* lds, int wave, int waves, F&& own) {
    const int lane = threadIdx.x & 63;
    constexpr int NP = NT / G;
    if (waves == 1) {
#pragma unroll
      for (int p = 0; p < NP; ++p)
#pragma unroll
        for (int f = 0; f < FR; ++f) {
          v4f y[G];
#pragma unroll
          for (int g = 0; g < G; ++g) y[g] = acc[p + g * NP][f];
          own(p, f, y);
        }
      return;
    }
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int f = 0; f < FR; ++f) lds[((wave * NT + n) * FR + f) * 64 + lane] = acc[n][f];
    __syncthreads();
    for (int i = wave; i < NP * FR; i += waves) {
      const int p = i / FR, f = i % FR;
      v4f y[G];
#pragma unroll
      for (int g = 0; g < G; ++g) {
        y[g] = lds[((p + g * NP) * FR + f) * 64 + lane];
        for (int k = 1; k < waves; ++k) y[g] += lds[((k * NT + p + g * NP) * FR + f) * 64 + lane];
      }
      own(p, f, y);
    }
  }
};

__device__ __forceinline__ uint32_t bf16_pair(float a, float b) {
  auto one = [](float v) -> uint32_t { return v == v ? bf16_rne(v) : 0x7FC0u; };
  return one(a) | one(b) << 16;
}

__device__ __forceinline__ int chunk_begin(int KC, int wave, int waves) { return KC * wave / waves; }

// Four outputs of row t from column n on.
__device__ __forceinline__ void store_linear(uint16_t* __restrict__ out, int t, int n, int N, const v4f& y) {
  if (n >= N) return;
  uint16_t* dst = out + (size_t)t * N + n;
  const uint32_t lo = bf16_pair(y[0], y[1]), hi = bf16_pair(y[2], y[3]);
  if ((N & 3) == 0) {
    *reinterpret_cast<uint2*>(dst) = make_uint2(lo, hi);
  } else {
    dst[0] = (uint16_t)lo;
    if (n + 1 < N) dst[1] = (uint16_t)(lo >> 16);
    if (n + 2 < N) dst[2] = (uint16_t)hi;
    if (n + 3 < N) dst[3] = (uint16_t)(hi >> 16);
  }
}

// y[t, n]: workgroup (row tiles nt*NT .., token group tg).
template <int NT, int FR>
__global__ void __launch_bounds__(512)
linear_w4_kernel(const uint8_t* __restrict__ x, const float* __restrict__ xs,
                                 const uint8_t* __restrict__ packed, int T, int N, int K,
                                 uint16_t* __restrict__ out) {
  extern __shared__ v4f s_part[];
  const int lane = threadIdx.x & 63, waves = blockDim.x >> 6;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int KC = w4_chunks(K), tiles = w4_tiles(N), KB = K / BLK;
  const int t0 = blockIdx.y * (16 * FR), n0 = blockIdx.x * NT;
  Stream<NT, FR> st;
#pragma unroll
  for (int n = 0; n < NT; ++n)
    st.w[n] = packed + (size_t)min(n0 + n, tiles - 1) * KC * W4_CHUNK_BYTES + lane * 16;
#pragma unroll
  for (int f = 0; f < FR; ++f) {
    const int t = min(t0 + 16 * f + (lane & 15), T - 1);  // padding columns reread the last row
    st.x[f] = x + (size_t)t * K + 16 * (lane >> 4);
    st.xs[f] = xs + t;
  }
  st.xs_stride = T;
  st.run(chunk_begin(KC, wave, waves), chunk_begin(KC, wave + 1, waves), KB);
  st.template reduce<1>(s_part, wave, waves, [&](int p, int f, const v4f* y) {
    const int t = t0 + 16 * f + (lane & 15);
    if (t < T) store_linear(out, t, (n0 + p) * 16 + 4 * (lane >> 4), N, y[0]);
  });
}

// ---------------------------------------------------------------------------
// Tiles, for many activation rows.  A workgroup of 4 waves multiplies 256 weight
// rows with up to 64 activation rows, two workgroups a CU: a wave takes 4 weight tiles
// and all the rows.  The weights go from global memory to the registers of the wave
// that owns their rows, three K-blocks ahead; the activations, which every wave
// needs, go through LDS, a step of two or four K-blocks ahead.  Per K-block a wave reads 2 KB
// of LDS for each four MFMAs (128 clocks of its SIMD): half of the LDS bandwidth with
// two waves a SIMD.  What bounds it: the MFMAs take 37% of the clocks and the scales'
// multiply-adds (four a product) and addresses another 40%, beside each other only where
// both waves of a SIMD have work.  T = 8192, N = 4096, K = 7168 in 244 us, 1.97 PFLOP/s
// (the library's FP8 product without scales reaches 2.56); T = 1501, N = 7168, K = 2048,
// two rounds of workgroups, in 33 us, 1.33.
//
// LDS rows are 128 bytes; the 16-byte piece q of row m lies at position q ^ (m & 7),
// so that eight lanes with eight consecutive rows read eight different banks' groups.
// ---------------------------------------------------------------------------
constexpr int TILE_ROWS = 256, TILE_THREADS = 256, TILE_MAX_NC = 5, TILE_WGS = 2;  // workgroups a CU
constexpr int TILE_COLS = 16, TILE_MAX_M = TILE_COLS * TILE_MAX_NC;                 // activation rows
// K-blocks of activations that are staged at once, between two barriers: four where they are
// few (N = 4096, K = 7168: T = 128 16.5 us with two, 14.9 with four; T = 256 19.7 and 16.7).
constexpr int step_blocks(int nc) { return nc <= 2 ? 4 : 2; }
constexpr int STEP_ROWS = 2 * TILE_MAX_M;  // rows times K-blocks of a step at most
static_assert(2 * TILE_COLS * step_blocks(2) <= STEP_ROWS, "a step of the small tiles");
struct TileLds {
  uint8_t x[2][STEP_ROWS * BLK];  // [K-block][row][128]
  float xs[2][STEP_ROWS];
  size_t row[TILE_MAX_M];  // byte offset of each activation row
  union {
    float amax[4][TILE_MAX_M];  // GEMM1
    struct {                    // GEMM2
      int token[TILE_MAX_M];
      float weight[TILE_MAX_M];
    };
  };
};
__device__ __forceinline__ uint32_t tile_slot(int row, int piece) {
  return (uint32_t)(row * BLK + ((piece ^ (row & 7)) << 4));
}

// acc[n][c]: the wave's 16 x 16 results.  row_of(m): the activation row of tile row
// m < 16 NC, of `K` bytes at x, its scales at xs + row * xs_row + kb * xs_block.
template <int NC, class RowOf>
__device__ __forceinline__ void tile_product(TileLds& s, const uint8_t* const (&w)[4], int K, const uint8_t* x,
                                             const float* xs, size_t xs_row, size_t xs_block, RowOf&& row_of,
                                             v4f (&acc)[4][NC]) {
  constexpr int M = TILE_COLS * NC, NR = W4_CHUNK_BLOCKS, NS = step_blocks(NC);
  constexpr int PIECES = NS * 8, PER = M * PIECES / TILE_THREADS;  // 16-byte pieces of a row's step, and per thread
  const int tid = threadIdx.x, lane = tid & 63, KB = K / BLK, last = (KB - 1) / NR;
  const v4f zero4 = {0.f, 0.f, 0.f, 0.f};
  // Thread tid fetches one piece of the step's K-blocks of rows tid / PIECES +
  // (TILE_THREADS / PIECES) i, and the scale of row tid % M, K-block tid / M.
  const int piece = tid % PIECES, row0 = tid / PIECES;
  const float* scale = xs + (size_t)row_of(tid % M) * xs_row + (size_t)(tid / M) * xs_block;
  if (tid < M) s.row[tid] = (size_t)row_of(tid) * K;
  constexpr bool IN_REGS = NC <= 2;  // the rows' addresses, else read again for each step
  const uint8_t* rows[IN_REGS ? PER : 1];
  auto row_at = [&](int i) __attribute__((always_inline)) {
    return x + s.row[row0 + i * (TILE_THREADS / PIECES)] + (piece & 7) * 16;
  };
  u32x4 st[PER];
  float ss = 0.0f;
  // Piece i of a step: its load (past the end of K: anything), and its write to LDS
  // (zeros there, which the padded weights need: a NaN code times zero is NaN).
  auto fetch = [&](int step, int i) __attribute__((always_inline)) {
    const int kb = step * NS + (piece >> 3);
    const uint8_t* row;
    if constexpr (IN_REGS) row = rows[i];
    else row = row_at(i);
    st[i] = *reinterpret_cast<const u32x4*>(row + (size_t)(kb < KB ? kb : 0) * BLK);
  };
  auto stage = [&](int step, int i) __attribute__((always_inline)) {
    if (step * NS + (piece >> 3) >= KB) st[i] = u32x4{0, 0, 0, 0};
    *reinterpret_cast<u32x4*>(s.x[step & 1] + (piece >> 3) * (M * BLK) +
                              tile_slot(row0 + i * (TILE_THREADS / PIECES), piece & 7)) = st[i];
  };
  auto fetch_scale = [&](int step) __attribute__((always_inline)) {
    ss = tid < M * NS && step * NS + tid / M < KB ? scale[(size_t)step * NS * xs_block] : 0.0f;
  };
  auto stage_scale = [&](int step) __attribute__((always_inline)) {
    if (tid < M * NS) s.xs[step & 1][tid] = ss;
  };
  u32x4 a[NR][4];
  int sc[4], sc_next[4];
  auto load_a = [&](int chunk, auto bc) __attribute__((always_inline)) {
    constexpr int b = decltype(bc)::value;
#pragma unroll
    for (int n = 0; n < 4; ++n)
      a[b][n] = *reinterpret_cast<const u32x4*>(w[n] + (size_t)chunk * W4_CHUNK_BYTES + (uint32_t)(b * W4_BLOCK_BYTES + lane * 16));
  };
  auto load_sc = [&](int chunk) __attribute__((always_inline)) {
#pragma unroll
    for (int n = 0; n < 4; ++n)
      sc_next[n] = *reinterpret_cast<const int*>(w[n] + (size_t)chunk * W4_CHUNK_BYTES +
                                                 (uint32_t)(W4_CHUNK_BLOCKS * W4_BLOCK_BYTES + lane * 4));
  };
#pragma unroll
  for (int n = 0; n < 4; ++n)
#pragma unroll
    for (int c = 0; c < NC; ++c) acc[n][c] = zero4;

  load_sc(0);
  load_a(0, std::integral_constant<int, 0>{});
  load_a(0, std::integral_constant<int, 1>{});
  load_a(0, std::integral_constant<int, 2>{});
  fetch_scale(0);
  __syncthreads();
  if constexpr (IN_REGS) {
#pragma unroll
    for (int i = 0; i < PER; ++i) rows[i] = row_at(i);
  }
#pragma unroll
  for (int i = 0; i < PER; ++i) fetch(0, i);
#pragma unroll
  for (int i = 0; i < PER; ++i) stage(0, i);
  stage_scale(0);
#pragma unroll
  for (int i = 0; i < PER; ++i) fetch(1, i);
  fetch_scale(1);
  __syncthreads();
  const int i16 = lane & 15, g = lane >> 4;
#pragma unroll 1
  for (int chunk = 0; chunk <= last; ++chunk) {
#pragma unroll
    for (int n = 0; n < 4; ++n) sc[n] = sc_next[n];
    static_for<NR / NS>([&](auto hc) __attribute__((always_inline)) {
      constexpr int h = decltype(hc)::value;
      const int step = chunk * (NR / NS) + h;
      const uint8_t* xb = s.x[step & 1];
      const float* xsb = s.xs[step & 1];
      // Fragment j of the step: K-block j / NC, rows 16 (j % NC) ..; its LDS reads run one
      // fragment ahead of its MFMAs.  Between the first half of the fragments the next
      // step's activations go to LDS (past the last: the buffer takes zeros), between
      // the second those of the step after it come in.
      u32x4 lo[2], hi[2];
      float sx[2];
      auto read = [&](auto jc) __attribute__((always_inline)) {
        constexpr int j = decltype(jc)::value, bb = j / NC, m0 = j % NC * 16;
        lo[j & 1] = *reinterpret_cast<const u32x4*>(xb + bb * (M * BLK) + tile_slot(m0 + i16, g));
        hi[j & 1] = *reinterpret_cast<const u32x4*>(xb + bb * (M * BLK) + tile_slot(m0 + i16, g + 4));
        sx[j & 1] = xsb[bb * M + m0 + i16];
      };
      read(std::integral_constant<int, 0>{});
      static_for<NS * NC>([&](auto jc) __attribute__((always_inline)) {
        constexpr int j = decltype(jc)::value, bb = h * NS + j / NC, c = j % NC;
        if constexpr (c == 0) {  // K-block bb + 3, into the slot that the last one used
          load_a(bb == 0 ? chunk : min(chunk + 1, last), std::integral_constant<int, (bb + 3) % NR>{});
          if constexpr (bb == 0) load_sc(min(chunk + 1, last));
        }
        if constexpr (j + 1 < NS * NC) read(std::integral_constant<int, j + 1>{});
        __builtin_amdgcn_sched_barrier(0);  // the reads stay ahead of this fragment's MFMAs
        const v8i xv = __builtin_bit_cast(v8i, __builtin_shufflevector(lo[j & 1], hi[j & 1], 0, 1, 2, 3, 4, 5, 6, 7));
#pragma unroll
        for (int n = 0; n < 4; ++n) {
          acc[n][c] += mfma_w4<bb>(a[bb][n], xv, sc[n], zero4) * sx[j & 1];
          // Keeps the addition here: the compiler would sink it to the loop's end, with the
          // products of the whole chunk in registers until then.
          __asm__ volatile("" : "+v"(acc[n][c]));
        }
        if constexpr (j < PER) stage(step + 1, j);
        if constexpr (j == PER - 1) {
          stage_scale(step + 1);
          fetch_scale(step + 2);
        }
        if constexpr (j >= PER) fetch(step + 2, j - PER);
      });
      __syncthreads();
    });
  }
}

// This workgroup's item of base .. n_work - 1, or -1.  They are cut into one run per XCD
// (workgroup b runs on XCD b % XCDS), so the items that share a route tile's
// activations share an L2.
__device__ __forceinline__ int xcd_item(int base, int n_work) {
  const int n = min(n_work - base, (int)gridDim.x), per = (n + XCDS - 1) / XCDS;
  const int q = blockIdx.x / XCDS, i = (int)(blockIdx.x % XCDS) * per + q;
  return q < per && i < n ? base + i : -1;
}
// The i-th item of nblk weight blocks x nt activation tiles: bands of up to 8 tiles, in a
// band block after block, so that the tiles that read one block's weights are neighbours,
// and a band's activations stay in the L2 from one block to the next.  (Weights of
// 131072 rows, T = 128, K = 7168: tile after tile 154 us, so 147; T = 1501, N = 7168,
// K = 2048: 34.8 and 32.0.)
__device__ __forceinline__ void banded(int i, int nblk, int nt, int& nb, int& tile) {
  constexpr int BAND = 8;
  const int band = i / (BAND * nblk), r = i - band * (BAND * nblk), width = min(BAND, nt - band * BAND);
  nb = r / width;
  tile = band * BAND + (r - nb * width);
}
// Launches for `items` items at most, each below 2^32 threads: f(grid, first item).
template <class F>
void by_grids(size_t items, F&& f) {
  for (size_t at = 0; at < items; at += MAX_GRID) {
    const size_t n = items - at < MAX_GRID ? items - at : MAX_GRID;
    f((unsigned)((n + XCDS - 1) / XCDS * XCDS), (int)at);
  }
}

template <int NC>
__global__ void __launch_bounds__(TILE_THREADS, TILE_WGS)
linear_w4_tile_kernel(const uint8_t* __restrict__ x, const float* __restrict__ xs, const uint8_t* __restrict__ packed,
                      int T, int N, int K, int base, uint16_t* __restrict__ out) {
  __shared__ __align__(16) TileLds s;
  const int tid = threadIdx.x, lane = tid & 63;
  const int rw = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int KC = w4_chunks(K), tiles = w4_tiles(N), blocks = (tiles + 15) / 16;
  const int token_tiles = (T + TILE_COLS * NC - 1) / (TILE_COLS * NC);
  const int item = xcd_item(base, blocks * token_tiles);
  if (item < 0) return;
  int nb, tt;
  banded(item, blocks, token_tiles, nb, tt);
  const int t0 = tt * (TILE_COLS * NC);
  const uint8_t* w[4];
#pragma unroll
  for (int n = 0; n < 4; ++n)
    w[n] = packed + (size_t)min(nb * 16 + rw * 4 + n, tiles - 1) * KC * W4_CHUNK_BYTES;
  v4f acc[4][NC];
  // Padding rows reread the last one.
  tile_product<NC>(s, w, K, x, xs, 1, T, [&](int m) { return min(t0 + m, T - 1); }, acc);
  // The results in bf16 through LDS, [row][256] with the 16-byte pieces spread as the
  // activations' are, so that 32 lanes store 512 contiguous bytes (straight from the
  // registers, 8 bytes a lane, the stores took 8 of 37 us at T = 1501, N = 7168, K = 2048).
  uint8_t* tile = s.x[0];
  constexpr int M = 16 * NC;
  static_assert(M * 512 <= (int)sizeof(s.x), "the tile in bf16");
  const int n0 = nb * TILE_ROWS;
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    const int m = c * 16 + (lane & 15);
#pragma unroll
    for (int n = 0; n < 4; ++n) {
      const int col = (rw * 4 + n) * 16 + 4 * (lane >> 4);  // of 256
      *reinterpret_cast<uint2*>(tile + m * 512 + (((col >> 3) ^ (m & 7)) << 4) + (col & 4) * 2) =
          make_uint2(bf16_pair(acc[n][c][0], acc[n][c][1]), bf16_pair(acc[n][c][2], acc[n][c][3]));
    }
  }
  __syncthreads();
  for (int i = tid; i < M * 32; i += TILE_THREADS) {
    const int m = i >> 5, q = i & 31, t = t0 + m, n = n0 + q * 8;
    if (t >= T || n >= N) continue;
    const u32x4 v = *reinterpret_cast<const u32x4*>(tile + m * 512 + ((q ^ (m & 7)) << 4));
    uint16_t* dst = out + (size_t)t * N + n;
    if ((N & 7) == 0) {
      *reinterpret_cast<u32x4*>(dst) = v;
    } else {
#pragma unroll
      for (int k = 0; k < 8; ++k)
        if (n + k < N) dst[k] = (uint16_t)(v[k >> 1] >> (16 * (k & 1)));
    }
  }
}

// ---------------------------------------------------------------------------
// The experts.  Dispatch: a counting sort of the local picks into routes, expert
// by expert, and a list of route tiles of `bm` routes.  A pick's place among its
// expert's routes is taken from an atomic and may differ from run to run; no
// result does, since every route is computed by itself and a token's routes are
// added in the order of its picks.
// ---------------------------------------------------------------------------
struct Routes {
  int32_t* offsets;      // [e_local + 1] first route of each expert; the last: their number
  int32_t* n_tiles;      // [1]
  int4* tiles;           // {expert, first route, routes, first tile of the expert}
  int32_t* tile_count;   // tiles of each tile's expert
  int32_t* route_token;  // [T k] token of each route; bit 31: its only local one
  float* route_weight;   // [T k]
  int32_t* pick_route;   // [T k], -1 for picks of other experts
  int32_t* chunk_counts; // [chunks][e_local]
};
// One launch sorts up to SORT_SMALL picks (its atomics on a few experts' counters take
// 3 ns a pick); more are cut into at most SORT_MAX_CHUNKS chunks of at least
// SORT_THREADS.
constexpr int SORT_THREADS = 1024, SORT_SMALL = 2048, SORT_MAX_CHUNKS = 64;
inline int sort_chunk(size_t picks) {
  const size_t per = (picks + SORT_MAX_CHUNKS - 1) / SORT_MAX_CHUNKS;
  return (int)((per + SORT_THREADS - 1) / SORT_THREADS * SORT_THREADS);
}
constexpr int MAX_EXPERTS = 1024;
constexpr int ONLY_BIT = (int)0x80000000u, TOKEN_MASK = 0x7FFFFFFF;

// s_scan[0 .. n) exclusive prefix sums of v over the threads; returns this
// thread's, `total` the sum.
__device__ __forceinline__ int block_scan(int v, int* s_wave, int& total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int inc = v;
  if (__any(v)) {  // most waves' experts are none
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int o = __shfl_up(inc, d);
      if (lane >= d) inc += o;
    }
  }
  __syncthreads();
  if (lane == 63) s_wave[wave] = inc;
  __syncthreads();
  int base = 0;
  total = 0;
  for (int w = 0; w < SORT_THREADS / 64; ++w) {
    base += w < wave ? s_wave[w] : 0;
    total += s_wave[w];
  }
  return base + inc - v;
}

// Routes per tile at most.  A launch of the tile kernels takes whole rounds of its items
// (tile, weight block) over the CUs, each about as long as its fragments of 32 routes and
// 1.2 more (K = 7168, 1 to 5 of them: 28, 34, 44, 60, 71 us a round); of the sizes the one
// with the shortest sum over GEMM1 (n1 weight blocks, k1 K-blocks) and GEMM2 is taken.
struct TilePlan {
  int bm;  // a fixed size, or 0: chosen
  int n1, k1, n2, k2;
  float per_cu;  // 1 / the workgroups that run at once
};

// Offsets and the tile list from expert `threadIdx.x`'s count: an expert's
// fragments of 16 routes, dealt evenly over as few tiles of at most bm routes as hold
// them.
__device__ __forceinline__ void publish_tiles(int cnt, int e_local, const TilePlan& plan, const Routes& r, int* s_off,
                                              int* s_tp, int* s_cnt, int* s_wave) {
  const int e = threadIdx.x;
  int total, tiles, bm = plan.bm;
  const int off = block_scan(cnt, s_wave, total);
  if (bm == 0) {
    // The sums of every size's tiles at once.
    constexpr int SIZES = TILE_MAX_NC - 1;
    __shared__ int s_sum[SIZES];
    if (e < SIZES) s_sum[e] = 0;
    __syncthreads();
    if (__any(cnt)) {
#pragma unroll
      for (int i = 0; i < SIZES; ++i) {
        const int m = (i + 2) * TILE_COLS;
        int n = (cnt + m - 1) / m;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) n += __shfl_xor(n, d);
        if ((e & 63) == 0) atomicAdd(&s_sum[i], n);
      }
    }
    __syncthreads();
    // Every lane the cost of size lane % SIZES, then all of them the least's (in equal
    // cases the largest) size.
    const int mine = e & (SIZES - 1);
    const float n = (float)max(s_sum[mine], 1);
    auto rounds = [&](int blocks) { return ceilf(n * (float)blocks * plan.per_cu - 1e-4f); };
    const float item = (float)total * __builtin_amdgcn_rcpf(TILE_COLS * n) + 1.2f;
    const float cost = item * (rounds(plan.n1) * (float)plan.k1 + rounds(plan.n2) * (float)plan.k2);
    float least = cost;
    int best = mine;
#pragma unroll
    for (int d = 1; d < SIZES; d <<= 1) {
      const float o = __shfl_xor(least, d);
      const int ob = __shfl_xor(best, d);
      if (o < least || (o == least && ob > best)) {
        least = o;
        best = ob;
      }
    }
    bm = (best + 2) * TILE_COLS;
  }
  const int tp = block_scan((cnt + bm - 1) / bm, s_wave, tiles);
  if (e < e_local) {
    s_off[e] = off;
    s_tp[e] = tp;
    s_cnt[e] = cnt;
    r.offsets[e] = off;
  }
  if (e == 0) {
    r.offsets[e_local] = total;
    *r.n_tiles = tiles;
  }
  __syncthreads();
  for (int i = e; i < tiles; i += SORT_THREADS) {
    int lo = 0, hi = e_local - 1;  // the last expert whose first tile is at most i: the one that has it
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (s_tp[mid] <= i) lo = mid;
      else hi = mid - 1;
    }
    const int n = s_cnt[lo], nt = (n + bm - 1) / bm;
    const int per = (((n + 15) >> 4) + nt - 1) / nt * 16, m0 = (i - s_tp[lo]) * per;
    r.tiles[i] = make_int4(lo, s_off[lo] + m0, min(per, n - m0), s_tp[lo]);
    r.tile_count[i] = nt;
  }
}

// Local expert of a pick, or -1.
__device__ __forceinline__ int local_expert(int id, int e_local, int offset) {
  const int e = id - offset;
  return id >= 0 && e >= 0 && e < e_local ? e : -1;
}

// Picks p0 .. p1 - 1 into their expert's places, from s_pos[e] on.
__device__ __forceinline__ void place_picks(const int32_t* __restrict__ ids, const float* __restrict__ weights, int p0, int p1, int k, int e_local,
                                            int offset, int* s_pos, const Routes& r) {
  for (int p = p0 + (int)threadIdx.x; p < p1; p += SORT_THREADS) {
    const int e = local_expert(ids[p], e_local, offset);
    int at = -1;
    if (e >= 0) {
      const int t = p / k;
      int n = 0;
      for (int j = t * k, j1 = j + k; j < j1; ++j) n += local_expert(ids[j], e_local, offset) >= 0 ? 1 : 0;
      at = atomicAdd(&s_pos[e], 1);
      r.route_token[at] = t | (n == 1 ? ONLY_BIT : 0);
      r.route_weight[at] = weights[p];
    }
    r.pick_route[p] = at;
  }
}
__device__ __forceinline__ void count_picks(const int32_t* __restrict__ ids, int p0, int p1, int e_local, int offset,
                                            int* s_cnt) {
  for (int p = p0 + (int)threadIdx.x; p < p1; p += SORT_THREADS) {
    const int e = local_expert(ids[p], e_local, offset);
    if (e >= 0) atomicAdd(&s_cnt[e], 1);
  }
}

// All picks, counted by both of two workgroups: the first publishes the offsets and the
// tiles, the second places the picks (512 of them: 6.7 us by one after the other, 4.7 so).
__global__ void __launch_bounds__(SORT_THREADS)
sort_small_kernel(const int32_t* __restrict__ ids, const float* __restrict__ weights, int picks, int k, int e_local, int offset, TilePlan plan, Routes r) {
  __shared__ int s_cnt[MAX_EXPERTS], s_off[MAX_EXPERTS], s_tp[MAX_EXPERTS], s_pos[MAX_EXPERTS], s_wave[16];
  const int tid = threadIdx.x;
  s_pos[tid] = 0;
  __syncthreads();
  count_picks(ids, 0, picks, e_local, offset, s_pos);
  __syncthreads();
  const int cnt = tid < e_local ? s_pos[tid] : 0;
  if (blockIdx.x == 0) {
    publish_tiles(cnt, e_local, plan, r, s_off, s_tp, s_cnt, s_wave);
    return;
  }
  int all;
  const int off = block_scan(cnt, s_wave, all);  // its barriers are behind everyone's reads
  s_pos[tid] = off;
  __syncthreads();
  place_picks(ids, weights, 0, picks, k, e_local, offset, s_pos, r);
}

// The same over several workgroups, `chunk` picks each: their counts, ...
__global__ void __launch_bounds__(SORT_THREADS)
sort_count_kernel(const int32_t* __restrict__ ids, int picks, int chunk, int e_local, int offset, Routes r) {
  __shared__ int s_cnt[MAX_EXPERTS];
  const int tid = threadIdx.x, p0 = blockIdx.x * chunk;
  s_cnt[tid] = 0;
  __syncthreads();
  count_picks(ids, p0, min(picks, p0 + chunk), e_local, offset, s_cnt);
  __syncthreads();
  if (tid < e_local) r.chunk_counts[(size_t)blockIdx.x * e_local + tid] = s_cnt[tid];
}
// ... and the places, behind those of the chunks before; one more workgroup publishes the
// offsets and the tiles meanwhile (T = 4001, 32008 picks: 12.5 us as two launches).
__global__ void __launch_bounds__(SORT_THREADS)
sort_place_kernel(const int32_t* __restrict__ ids, const float* __restrict__ weights, int picks, int chunk, int chunks, int k,
                  int e_local, int offset, TilePlan plan, Routes r) {
  __shared__ int s_cnt[MAX_EXPERTS], s_off[MAX_EXPERTS], s_pos[MAX_EXPERTS], s_wave[16];
  const int tid = threadIdx.x, me = blockIdx.x;
  int total = 0, before = 0;  // expert tid's picks, and those of the chunks before this one
  if (tid < e_local) {
#pragma unroll 16
    for (int c = 0; c < chunks; ++c) {
      const int n = r.chunk_counts[(size_t)c * e_local + tid];
      total += n;
      before += c < me ? n : 0;
    }
  }
  if (me == chunks) {
    publish_tiles(total, e_local, plan, r, s_off, s_pos, s_cnt, s_wave);
    return;
  }
  int all;
  const int off = block_scan(total, s_wave, all);
  if (tid < e_local) s_pos[tid] = off + before;
  __syncthreads();
  place_picks(ids, weights, me * chunk, min(picks, (me + 1) * chunk), k, e_local, offset, s_pos, r);
}

// A route tile's entry, the same for all lanes: the weights' addresses stay in scalar
// registers.
__device__ __forceinline__ int4 uniform(const int4& t) {
  return make_int4(__builtin_amdgcn_readfirstlane(t.x), __builtin_amdgcn_readfirstlane(t.y),
                   __builtin_amdgcn_readfirstlane(t.z), __builtin_amdgcn_readfirstlane(t.w));
}

__device__ __forceinline__ float4 swiglu(const v4f& gate, const v4f& up) {
  auto one = [&](int i) { return up[i] / (1.0f + __expf(-up[i])) * gate[i]; };
  return make_float4(one(0), one(1), one(2), one(3));
}

// f(the fragments of 16 that hold `rows`, MAX at most).
template <int MAX, int N = 1, class F>
__device__ __forceinline__ void by_frags(int rows, F&& f) {
  if constexpr (N < MAX) {
    if (rows > 16 * N) return by_frags<MAX, N + 1>(rows, f);
  }
  f(std::integral_constant<int, N>{});
}

// GEMM1 and SwiGLU of (route tile, 16 gate and 16 up rows): rows
// [0, I) of W13 multiply, SiLU takes rows [I, 2 I).  Workgroups past the last
// tile end at once.  Bound by the weights' stream where most experts have routes (32 of
// them, T = 32: whole call 111 us for 749 MB of weights, 6.7 TB/s), and where few do by
// the activations' from the L2, 16 routes' or 32 for every 32 weight rows.
template <int MAXFR>
__global__ void __launch_bounds__(512)
experts_gemm1_kernel(ExpertsW4 a, Routes r, float* __restrict__ Cf) {
  extern __shared__ v4f s_part[];
  const int slices = a.I / 16;
  const int j = blockIdx.x % slices, n_tiles = *r.n_tiles;
  const int lane = threadIdx.x & 63, waves = blockDim.x >> 6;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int KC = w4_chunks(a.H), KB = a.H / BLK, tiles = 2 * a.I / 16;
  for (int i = blockIdx.x / slices; i < n_tiles; i += gridDim.x / slices) {
    if (i >= (int)(gridDim.x / slices)) __syncthreads();  // the waves have read the last tile's parts
    const int4 tile = uniform(r.tiles[i]);
    by_frags<MAXFR>(tile.z, [&](auto frc) __attribute__((always_inline)) {
      constexpr int FR = decltype(frc)::value;
      Stream<2, FR> st;
#pragma unroll
      for (int n = 0; n < 2; ++n) {
        st.w[n] = a.w13 + ((size_t)tile.x * tiles + j + n * slices) * KC * W4_CHUNK_BYTES + lane * 16;
      }
#pragma unroll
      for (int f = 0; f < FR; ++f) {
        const int t = r.route_token[tile.y + min(16 * f + (lane & 15), tile.z - 1)] & TOKEN_MASK;
        st.x[f] = a.x + (size_t)t * a.H + 16 * (lane >> 4);
        st.xs[f] = a.xs + t;
      }
      st.xs_stride = a.T;
      st.run(chunk_begin(KC, wave, waves), chunk_begin(KC, wave + 1, waves), KB);
      st.template reduce<2>(s_part, wave, waves, [&](int, int f, const v4f* y) {
        const int m = 16 * f + (lane & 15);
        if (m >= tile.z) return;
        *reinterpret_cast<float4*>(Cf + (size_t)(tile.y + m) * a.I + j * 16 + 4 * (lane >> 4)) =
            swiglu(y[0], y[1]);
      });
    });
  }
}

// Four columns of a route's W2 c, times its weight: to Y, or to the output row of a
// token that has no other local pick.
__device__ __forceinline__ void store_y(const ExpertsW4& a, float* __restrict__ Y, int route, int token, float weight,
                                        int col, const v4f& v) {
  const v4f y = v * weight;
  if (token < 0)  // 0 + y, as the combine's sum of one: -0 becomes +0
    *reinterpret_cast<uint2*>(a.out + (size_t)(token & TOKEN_MASK) * a.H + col) =
        make_uint2(bf16_pair(y[0] + 0.0f, y[1] + 0.0f), bf16_pair(y[2] + 0.0f, y[3] + 0.0f));
  else
    *reinterpret_cast<float4*>(Y + (size_t)route * a.H + col) = make_float4(y[0], y[1], y[2], y[3]);
}

// GEMM2 of (route tile, NT 16-row tiles of W2), times the pick's weight.
template <int NT, int MAXFR>
__global__ void __launch_bounds__(512)
experts_gemm2_kernel(ExpertsW4 a, Routes r, const uint8_t* __restrict__ Cq,
                                     const float* __restrict__ Cs, float* __restrict__ Y) {
  extern __shared__ v4f s_part[];
  const int slices = a.H / 16 / NT;
  const int j = blockIdx.x % slices, n_tiles = *r.n_tiles;
  const int lane = threadIdx.x & 63, waves = blockDim.x >> 6;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int KC = w4_chunks(a.I), KB = a.I / BLK, tiles = a.H / 16;
  for (int i = blockIdx.x / slices; i < n_tiles; i += gridDim.x / slices) {
    if (i >= (int)(gridDim.x / slices)) __syncthreads();  // the waves have read the last tile's parts
    const int4 tile = uniform(r.tiles[i]);
    by_frags<MAXFR>(tile.z, [&](auto frc) __attribute__((always_inline)) {
      constexpr int FR = decltype(frc)::value;
      Stream<NT, FR> st;
#pragma unroll
      for (int n = 0; n < NT; ++n)
        st.w[n] = a.w2 + ((size_t)tile.x * tiles + j * NT + n) * KC * W4_CHUNK_BYTES + lane * 16;
#pragma unroll
      for (int f = 0; f < FR; ++f) {
        const size_t row = tile.y + min(16 * f + (lane & 15), tile.z - 1);
        st.x[f] = Cq + row * a.I + 16 * (lane >> 4);
        st.xs[f] = Cs + row * KB;
      }
      st.xs_stride = 1;
      st.run(chunk_begin(KC, wave, waves), chunk_begin(KC, wave + 1, waves), KB);
      st.template reduce<1>(s_part, wave, waves, [&](int p, int f, const v4f* y) {
        const int m = 16 * f + (lane & 15);
        if (m >= tile.z) return;
        store_y(a, Y, tile.y + m, r.route_token[tile.y + m], r.route_weight[tile.y + m], (j * NT + p) * 16 + 4 * (lane >> 4),
                y[0]);
      });
    });
  }
}

// ---------------------------------------------------------------------------
// At most 64 picks in all: every workgroup sorts them itself, one per lane, and GEMM2
// requantises and combines, so a call is two launches (T = 1: 26 us with the five of
// the general path, whose kernels take 3 us each for nothing but their launch).  T = 1, one local pick's 23 MB:
// 7.0 and 4.9 us, which latency bounds (the picks, then the weights).
// Rows of Cf are picks here.
// ---------------------------------------------------------------------------
constexpr int FEW_PICKS = 64;
struct FewLds {
  int pick[FEW_PICKS], expert[FEW_PICKS];  // the local picks, by expert, then pick
};
struct FewTile {
  int expert, first, rows;  // rows places of FewLds::pick from `first` on
};
// Sorts the picks; returns a mask whose bits are the tiles' first places (tiles of at
// most 16 routes of one expert), and the number of local picks in n.  Every wave calls it.
__device__ __forceinline__ uint64_t few_sort(const ExpertsW4& a, FewLds& s, int& n) {
  const int lane = threadIdx.x & 63, picks = a.T * a.k;
  const int e = lane < picks ? local_expert(a.ids[lane], a.e_local, a.offset) : -1;
  const uint64_t local = __ballot(e >= 0);
  n = __popcll(local);
  int rank = 0;
  for (uint64_t m = local; m; m &= m - 1) {
    const int q = __builtin_ctzll(m), o = __builtin_amdgcn_readlane(e, q);
    rank += o < e || (o == e && q < lane) ? 1 : 0;
  }
  if (e >= 0) {  // all waves write the same
    s.pick[rank] = lane;
    s.expert[rank] = e;
  }
  __syncthreads();
  const int mine = lane < n ? s.expert[lane] : -1, before = lane > 0 && lane < n ? s.expert[lane - 1] : -2;
  const uint64_t starts = __ballot(lane < n && mine != before);
  // the place within the expert's run: from the last start at or below this lane
  const uint64_t below = starts & (~0ull >> (63 - lane));
  const int from = below ? 63 - __builtin_clzll(below) : 0;
  return __ballot(lane < n && ((lane - from) & 15) == 0);
}
__device__ __forceinline__ FewTile few_tile(const FewLds& s, uint64_t tiles, int i, int n) {
  for (int j = 0; j < i; ++j) tiles &= tiles - 1;
  const int first = __builtin_ctzll(tiles);
  tiles &= tiles - 1;
  return {s.expert[first], first, (tiles ? __builtin_ctzll(tiles) : n) - first};
}

// GEMM1 and SwiGLU of (tile, 16 gate and 16 up rows).
__global__ void __launch_bounds__(512)
few_gemm1_kernel(ExpertsW4 a, float* __restrict__ Cf) {
  extern __shared__ v4f s_part[];
  __shared__ FewLds s;
  const int slices = a.I / 16, i = blockIdx.x / slices, j = blockIdx.x % slices;
  int n;
  const uint64_t tiles = few_sort(a, s, n);
  if (i >= __popcll(tiles)) return;
  const FewTile tile = few_tile(s, tiles, i, n);
  const int lane = threadIdx.x & 63, waves = blockDim.x >> 6;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int KC = w4_chunks(a.H), expert = __builtin_amdgcn_readfirstlane(tile.expert);
  Stream<2, 1> st;
#pragma unroll
  for (int g = 0; g < 2; ++g)
    st.w[g] = a.w13 + ((size_t)expert * (2 * slices) + g * slices + j) * KC * W4_CHUNK_BYTES + lane * 16;
  const int t = s.pick[tile.first + min(lane & 15, tile.rows - 1)] / a.k;
  st.x[0] = a.x + (size_t)t * a.H + 16 * (lane >> 4);
  st.xs[0] = a.xs + t;
  st.xs_stride = a.T;
  st.run(chunk_begin(KC, wave, waves), chunk_begin(KC, wave + 1, waves), a.H / BLK);
  st.reduce<2>(s_part, wave, waves, [&](int, int, const v4f* y) {
    if ((lane & 15) >= tile.rows) return;
    *reinterpret_cast<float4*>(Cf + (size_t)s.pick[tile.first + (lane & 15)] * a.I + j * 16 + 4 * (lane >> 4)) =
        swiglu(y[0], y[1]);
  });
}

// GEMM2 of 32 output columns of every token: per tile the workgroup requantises its
// rows of Cf into LDS (each of the H / 32 workgroups does: 2048 elements a route), wave
// (nt, cw) multiplies weight tile nt with chunks cw, cw + 4, ..., the parts are added in K
// order, and the picks' results, times their weights, are kept until all are there.
constexpr int FEW_THREADS = 512, FEW_MAX_I = 2048;
__global__ void __launch_bounds__(FEW_THREADS)
few_gemm2_kernel(ExpertsW4 a, const float* __restrict__ Cf) {
  extern __shared__ __align__(16) uint8_t s_x[];  // codes [16][I], 16-byte pieces at piece ^ (row & 7)
  __shared__ FewLds s;
  __shared__ float s_xs[16][FEW_MAX_I / BLK];
  __shared__ v4f s_part[8][64];
  __shared__ float s_y[FEW_PICKS][33];
  int n;
  uint64_t tiles = few_sort(a, s, n);
  const int tid = threadIdx.x, lane = tid & 63, nt = __builtin_amdgcn_readfirstlane(tid >> 8);
  const int cw = __builtin_amdgcn_readfirstlane((tid >> 6) & 3), i16 = lane & 15, g = lane >> 4;
  const int KC = w4_chunks(a.I), KB = a.I / BLK, n_tiles = __popcll(tiles);
  const v4f zero4 = {0.f, 0.f, 0.f, 0.f};
  u32x4 w[4];
  int sc = 0;
  auto load = [&](int expert, int c) {
    const uint8_t* p = a.w2 + (((size_t)expert * (a.H / 16) + blockIdx.x * 2 + nt) * KC + c) * W4_CHUNK_BYTES;
#pragma unroll
    for (int b = 0; b < 4; ++b)
      w[b] = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(p + (uint32_t)(b * W4_BLOCK_BYTES + lane * 16)));
    sc = __builtin_nontemporal_load(
        reinterpret_cast<const int*>(p + (uint32_t)(W4_CHUNK_BLOCKS * W4_BLOCK_BYTES + lane * 4)));
  };
  for (int i = 0; i < n_tiles; ++i) {
    const FewTile tile = few_tile(s, tiles, 0, n);
    tiles &= tiles - 1;
    const int expert = __builtin_amdgcn_readfirstlane(tile.expert);
    if (cw < KC) load(expert, cw);  // in flight over the requantisation
    for (int u = tid >> 4; u < tile.rows * KB; u += FEW_THREADS / 16) {
      const int m = u / KB, kb = u - m * KB, sub = tid & 15;
      float f[8], scale;
      load8<DT_F32>(Cf, (size_t)s.pick[tile.first + m] * a.I + kb * BLK + sub * 8, f);
      const uint2 o = quant8(f, scale);
      *reinterpret_cast<uint2*>(s_x + m * a.I + kb * BLK + (((sub >> 1) ^ (m & 7)) << 4) + (sub & 1) * 8) = o;
      if (sub == 0) s_xs[m][kb] = scale;
    }
    __syncthreads();
    v4f acc = zero4;
    const int m = min(i16, tile.rows - 1);
    for (int c = cw; c < KC; c += 4) {
      if (c > cw) load(expert, c);
      static_for<4>([&](auto bc) __attribute__((always_inline)) {
        constexpr int b = decltype(bc)::value;
        const int kb = c * W4_CHUNK_BLOCKS + b;
        if (kb < KB) {
          const uint8_t* xb = s_x + m * a.I + kb * BLK;
          const u32x4 lo = *reinterpret_cast<const u32x4*>(xb + ((g ^ (m & 7)) << 4));
          const u32x4 hi = *reinterpret_cast<const u32x4*>(xb + (((g + 4) ^ (m & 7)) << 4));
          const v8i x = __builtin_bit_cast(v8i, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
          acc += mfma_w4<b>(w[b], x, sc, zero4) * s_xs[m][kb];
        }
      });
    }
    s_part[nt * 4 + cw][lane] = acc;
    __syncthreads();
    if (tid < 128) {  // threads (nt, lane): the four columns of one route
      const int h = tid >> 6;
      v4f y = s_part[h * 4][lane];
      for (int c = 1; c < 4; ++c) y += s_part[h * 4 + c][lane];
      if (i16 < tile.rows) {
        const int p = s.pick[tile.first + i16];
        y *= a.weights[p];
#pragma unroll
        for (int v = 0; v < 4; ++v) s_y[p][h * 16 + 4 * g + v] = y[v];
      }
    }
  }
  __syncthreads();
  for (int i = tid; i < a.T * 16; i += FEW_THREADS) {
    const int t = i >> 4, col = (i & 15) * 2;
    float y0 = 0.0f, y1 = 0.0f;
    for (int p = t * a.k; p < (t + 1) * a.k; ++p)
      if (local_expert(a.ids[p], a.e_local, a.offset) >= 0) {
        y0 += s_y[p][col];
        y1 += s_y[p][col + 1];
      }
    *reinterpret_cast<uint32_t*>(a.out + (size_t)t * a.H + blockIdx.x * 32 + col) = bf16_pair(y0, y1);
  }
}

// The experts' products in tiles (route tiles of at most TILE_MAX_M).  f(NC) for
// the fewest fragments that hold `rows`.
template <int NC = 1, class F>
__device__ __forceinline__ void by_rows(int rows, F&& f) {
  if constexpr (NC < TILE_MAX_NC) {
    if (rows > TILE_COLS * NC) return by_rows<NC + 1>(rows, f);
  }
  f(std::integral_constant<int, NC>{});
}

// The tile and weight block of an item: experts in turn, an expert's items banded.
__device__ __forceinline__ int4 expert_item(const Routes& r, int item, int nblk, int& nb) {
  const int i = item / nblk, first = __builtin_amdgcn_readfirstlane(r.tiles[i].w);
  int tile;
  banded(item - first * nblk, nblk, __builtin_amdgcn_readfirstlane(r.tile_count[i]), nb, tile);
  return uniform(r.tiles[first + tile]);
}

// GEMM1, SwiGLU and the FP8 requantisation of (route tile, 128 columns of the
// intermediate): wave rw's weight tiles are 32 gate and the same 32 up rows.  7168, 2048,
// 32 of 256 experts, T = 4001: 164 us, 1.4 PFLOP/s; GEMM2 106 us, 1.1 with its fp32 rows.
// T = 64 on six experts: 28 us for 94 MB, which 96 workgroups' loads bound (a CU streams
// 35 to 65 GB/s, however far ahead it loads).
__global__ void __launch_bounds__(TILE_THREADS, TILE_WGS)
experts_gemm1_tile_kernel(ExpertsW4 a, Routes r, int base, uint8_t* __restrict__ Cq, float* __restrict__ Cs) {
  __shared__ __align__(16) TileLds s;
  const int IB = a.I / BLK;
  const int item = xcd_item(base, *r.n_tiles * IB);
  if (item < 0) return;
  int nb;
  const int4 tile = expert_item(r, item, IB, nb);
  const int tid = threadIdx.x, lane = tid & 63, g = lane >> 4;
  const int rw = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int KC = w4_chunks(a.H), tiles = 2 * a.I / 16;
  const uint8_t* w[4];
#pragma unroll
  for (int n = 0; n < 4; ++n) {
    const int row = nb * 8 + 2 * rw + (n & 1) + (n >> 1) * (a.I / 16);
    w[n] = a.w13 + ((size_t)tile.x * tiles + row) * KC * W4_CHUNK_BYTES;
  }
  by_rows(tile.z, [&](auto ncc) __attribute__((always_inline)) {
    constexpr int NC = decltype(ncc)::value;
    v4f acc[4][NC];
    tile_product<NC>(s, w, a.H, a.x, a.xs, 1, a.T, [&](int m) {
      return r.route_token[tile.y + min(m, tile.z - 1)] & TOKEN_MASK;
    }, acc);
    // c in place of the gate's results, and the waves' largest magnitudes per route.
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      float mx = 0.0f;
#pragma unroll
      for (int p = 0; p < 2; ++p)
#pragma unroll
        for (int v = 0; v < 4; ++v) {
          const float up = acc[2 + p][c][v];
          acc[p][c][v] *= up / (1.0f + __expf(-up));
          mx = fmaxf(mx, fabsf(acc[p][c][v]));
        }
      mx = fmaxf(mx, __shfl_xor(mx, 16));
      mx = fmaxf(mx, __shfl_xor(mx, 32));
      if (g == 0) s.amax[rw][c * 16 + lane] = mx;
    }
    __syncthreads();
    uint8_t* codes = s.x[0];
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      const int m = c * 16 + (lane & 15);
      float qs, qy;
      const float sc = block_scale(fmaxf(fmaxf(s.amax[0][m], s.amax[1][m]), fmaxf(s.amax[2][m], s.amax[3][m])), qs, qy);
#pragma unroll
      for (int p = 0; p < 2; ++p)
        *reinterpret_cast<uint32_t*>(codes + tile_slot(m, 2 * rw + p) + 4 * g) =
            quot4_e4m3(acc[p][c][0], acc[p][c][1], acc[p][c][2], acc[p][c][3], qs, qy);
      if (rw == 0 && g == 0 && m < tile.z) Cs[(size_t)(tile.y + m) * IB + nb] = sc;
    }
    __syncthreads();
    for (int i = tid; i < tile.z * 8; i += TILE_THREADS)
      *reinterpret_cast<u32x4*>(Cq + (size_t)(tile.y + (i >> 3)) * a.I + nb * BLK + (i & 7) * 16) =
          *reinterpret_cast<const u32x4*>(codes + tile_slot(i >> 3, i & 7));
  });
}

// GEMM2 of (route tile, 256 columns of the output; the last block may have 128).
__global__ void __launch_bounds__(TILE_THREADS, TILE_WGS)
experts_gemm2_tile_kernel(ExpertsW4 a, Routes r, int base, const uint8_t* __restrict__ Cq,
                          const float* __restrict__ Cs, float* __restrict__ Y) {
  __shared__ __align__(16) TileLds s;
  const int tiles = a.H / 16, blocks = (tiles + 15) / 16, KB = a.I / BLK;
  const int item = xcd_item(base, *r.n_tiles * blocks);
  if (item < 0) return;
  int nb;
  const int4 tile = expert_item(r, item, blocks, nb);
  const int tid = threadIdx.x, lane = tid & 63;
  const int rw = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int KC = w4_chunks(a.I);
  const uint8_t* w[4];
#pragma unroll
  for (int n = 0; n < 4; ++n)
    w[n] = a.w2 + ((size_t)tile.x * tiles + min(nb * 16 + rw * 4 + n, tiles - 1)) * KC * W4_CHUNK_BYTES;
  if (tid < TILE_MAX_M) {  // for the epilogue, behind the product's barriers
    s.token[tid] = r.route_token[tile.y + min(tid, tile.z - 1)];
    s.weight[tid] = r.route_weight[tile.y + min(tid, tile.z - 1)];
  }
  by_rows(tile.z, [&](auto ncc) __attribute__((always_inline)) {
    constexpr int NC = decltype(ncc)::value;
    v4f acc[4][NC];
    tile_product<NC>(s, w, a.I, Cq, Cs, KB, 1, [&](int m) { return tile.y + min(m, tile.z - 1); }, acc);
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      const int m = c * 16 + (lane & 15);
      if (m >= tile.z) continue;
      const int token = s.token[m];
      const float weight = s.weight[m];
#pragma unroll
      for (int n = 0; n < 4; ++n) {
        const int row = nb * 16 + rw * 4 + n;
        if (row < tiles) store_y(a, Y, tile.y + m, token, weight, row * 16 + 4 * (lane >> 4), acc[n][c]);
      }
    }
  });
}

// out[t] = the sum of its local picks' Y rows, in the order of the picks, where it
// has not just one.  Bound by the copy.
__global__ void __launch_bounds__(256)
experts_combine_kernel(const float* __restrict__ Y, const int32_t* __restrict__ pick_route, int H, int k,
                       uint16_t* __restrict__ out) {
  const int t = blockIdx.x, c = (blockIdx.y * 256 + threadIdx.x) * 4;
  if (c >= H) return;
  int n = 0;
  for (int j = 0; j < k; ++j) n += pick_route[(size_t)t * k + j] >= 0 ? 1 : 0;
  if (n == 1) return;  // GEMM2 has written it
  float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int j = 0; j < k; ++j) {
    const int r = pick_route[(size_t)t * k + j];
    if (r < 0) continue;
    const float4 y = *reinterpret_cast<const float4*>(Y + (size_t)r * H + c);
    s.x += y.x; s.y += y.y; s.z += y.z; s.w += y.w;
  }
  *reinterpret_cast<uint2*>(out + (size_t)t * H + c) = make_uint2(bf16_pair(s.x, s.y), bf16_pair(s.z, s.w));
}

struct ExpertsLayout {
  size_t offsets, n_tiles, tiles, tile_count, route_token, route_weight, pick_route, chunk_counts, cf, cq, cs, y, total;
};
// The smallest route tile sets the length of the tile list.
constexpr int MIN_BM = 16;
size_t max_tiles(size_t picks, int e_local, int bm) {
  return (picks < (size_t)e_local ? picks : (size_t)e_local) + picks / bm;
}
ExpertsLayout experts_layout(int T, int H, int I, int e_local, int k) {
  const size_t picks = (size_t)T * k, chunks = SORT_MAX_CHUNKS;
  size_t at = 0;
  auto take = [&](size_t bytes) {
    const size_t here = at;
    at += (bytes + 255) / 256 * 256;
    return here;
  };
  ExpertsLayout l;
  l.offsets = take(((size_t)e_local + 1) * 4);
  l.n_tiles = take(4);
  l.tiles = take(max_tiles(picks, e_local, MIN_BM) * 16);
  l.tile_count = take(max_tiles(picks, e_local, MIN_BM) * 4);
  l.route_token = take(picks * 4);
  l.route_weight = take(picks * 4);
  l.pick_route = take(picks * 4);
  l.chunk_counts = take(chunks * e_local * 4);
  l.cf = take(picks * I * 4);
  l.cq = take(picks * I);
  l.cs = take(picks * (I / BLK) * 4);
  l.y = take(picks * H * 4);
  l.total = at;
  return l;
}

}  // namespace

size_t w4_packed_bytes(int N, int K) { return (size_t)w4_tiles(N) * w4_chunks(K) * W4_CHUNK_BYTES; }

hipError_t launch_pack_w4(uint8_t* codes, uint8_t* scales, uint8_t* packed, int n, int N, int K, bool unpack,
                          hipStream_t stream) {
  const size_t units = (size_t)n * w4_tiles(N) * w4_chunks(K) * W4_CHUNK_BLOCKS * 64;
  pack_w4_kernel<<<(unsigned)((units + 255) / 256), 256, 0, stream>>>(codes, scales, packed, N, K, units, unpack);
  return hipGetLastError();
}

hipError_t launch_quantize_w4(const void* w, int dtype, size_t groups, uint8_t* codes, uint8_t* scales,
                              hipStream_t stream) {
  const unsigned grid = (unsigned)((groups * 4 + 255) / 256);
  if (dtype == DT_F32) quantize_w4_kernel<DT_F32><<<grid, 256, 0, stream>>>(w, groups, codes, scales);
  else if (dtype == DT_BF16) quantize_w4_kernel<DT_BF16><<<grid, 256, 0, stream>>>(w, groups, codes, scales);
  else quantize_w4_kernel<DT_F16><<<grid, 256, 0, stream>>>(w, groups, codes, scales);
  return hipGetLastError();
}

hipError_t launch_quant_act(const void* x, int dtype, size_t row_stride, int T, int K, uint8_t* codes, float* scale,
                            hipStream_t stream) {
  const int KB = K / BLK, rows = (T + 15) / 16;
  auto launch = [&](auto dt) {
    constexpr int DT = decltype(dt)::value;
    // Four blocks a thread where that leaves two workgroups a CU (T = 8192, K = 7168:
    // 48 us with one of whole rows' blocks in turn, 38 with four).
    if ((size_t)rows * ((KB + 3) / 4) >= 2 * (size_t)device_cus())
      quant_act_kernel<DT, 4><<<dim3(rows, (KB + 3) / 4), 256, 0, stream>>>(x, row_stride, T, KB, codes, scale);
    else
      quant_act_kernel<DT, 1><<<dim3(rows, KB), 256, 0, stream>>>(x, row_stride, T, KB, codes, scale);
  };
  if (dtype == DT_F32) launch(std::integral_constant<int, DT_F32>{});
  else if (dtype == DT_BF16) launch(std::integral_constant<int, DT_BF16>{});
  else launch(std::integral_constant<int, DT_F16>{});
  return hipGetLastError();
}

// Whether a dense product runs in tiles.  A tile launch of few items takes its K loop's
// time, a stream's time goes with the outputs; us, tiles / streams:
//   N=4096 K=7168  T=64 20.6 / 12.6, 96 20.3 / 20.1, 128 20.1 / 20.6, 192 20.4 / 30.2
//   N=2048 K=4096  T=128 9.8 / 8.3, 192 10.2 / 12.6
//   N=7168 K=2048  T=32 7.0 / 6.4, 33 7.0 / 7.4, 128 7.3 / 12.9
//   N=2000 K=512   T=64 4.2 / 4.5, 128 4.2 / 4.9
//   N=1024 K=1024  T=256 4.9 / 4.6;  N=512 K=7168  T=256 14.4 / 11.7
static bool linear_in_tiles(int T, int N, int K) { return (size_t)T * N > 150000 + 45 * (size_t)K; }

// Fragments per wave of a tile launch: the fewest whole rounds of workgroups over
// the CUs, each as long as its fragments and a constant share (weights, barriers).
static int linear_tile_nc(int T, int tiles, int cus) {
  int best = 1;
  float least = 0.0f;
  for (int nc = 1; nc <= TILE_MAX_NC; ++nc) {
    const long long items = (long long)((tiles + 15) / 16) * ((T + TILE_COLS * nc - 1) / (TILE_COLS * nc));
    const float cost = (float)((items + cus - 1) / cus) * (nc + 1.2f);
    if (nc == 1 || cost < least) { best = nc; least = cost; }
  }
  return best;
}

// Waves that share KC chunks: up to 8, each with as many but for the last.
static int stream_waves(int KC) {
  const int per = (KC + 7) / 8;
  return (KC + per - 1) / per;
}

hipError_t launch_linear_w4(const uint8_t* x, const float* xs, const uint8_t* packed, int T, int N, int K,
                            uint16_t* out, hipStream_t stream) {
  const int tiles = w4_tiles(N), KC = w4_chunks(K);
  const int waves = stream_waves(KC);
  if (linear_in_tiles(T, N, K)) {
    auto tile = [&](auto kernel, int nc) {
      const size_t items = (size_t)((tiles + 15) / 16) * ((T + TILE_COLS * nc - 1) / (TILE_COLS * nc));
      by_grids(items, [&](unsigned grid, int base) {
        kernel<<<grid, TILE_THREADS, 0, stream>>>(x, xs, packed, T, N, K, base, out);
      });
    };
    switch (linear_tile_nc(T, tiles, device_cus() * TILE_WGS)) {
      case 1: tile(linear_w4_tile_kernel<1>, 1); break;
      case 2: tile(linear_w4_tile_kernel<2>, 2); break;
      case 3: tile(linear_w4_tile_kernel<3>, 3); break;
      case 4: tile(linear_w4_tile_kernel<4>, 4); break;
      default: tile(linear_w4_tile_kernel<5>, 5); break;
    }
    return hipGetLastError();
  }
  auto launch = [&](auto kernel, int nt, int fr) {
    const dim3 grid((tiles + nt - 1) / nt, (T + 16 * fr - 1) / (16 * fr));
    kernel<<<grid, 64 * waves, waves > 1 ? waves * nt * fr * 1024 : 0, stream>>>(x, xs, packed, T, N, K, out);
  };
  if (T <= 16) launch(linear_w4_kernel<1, 1>, 1, 1);
  else launch(linear_w4_kernel<2, 2>, 2, 2);
  return hipGetLastError();
}

// Whether the experts' products run in tiles: from 49 tokens on where a tile per
// expert fills the CUs, else from 385 on.  Whole call, us, tiles / streams:
//   7168, 2048, 32 of 256, top 8   even T=32 108 / 111, 64 126 / 137, 128 143 / 160, 512
//     167 / 249; uneven T=32 50 / 45, 64 54 / 58, 128 58 / 79, 512 87 / 186
//   2048, 768, 128 of 128, top 8   even T=32 69 / 74, 64 78 / 84, 512 109 / 177
//   1024, 512, 16 of 64, top 4 (64 items)   even T=64 19 / 18, 256 23 / 22, 512 25 / 26
static bool experts_in_tiles(const ExpertsW4& a) {
  return a.T > ((long long)a.e_local * (a.I / BLK) >= device_cus() ? 48 : 384);
}

size_t experts_w4_workspace(int T, int H, int I, int e_local, int k) {
  return experts_layout(T, H, I, e_local, k).total;
}

hipError_t launch_experts_w4(const ExpertsW4& a, uint8_t* ws, hipStream_t stream) {
  const ExpertsLayout l = experts_layout(a.T, a.H, a.I, a.e_local, a.k);
  auto i32 = [&](size_t at) { return reinterpret_cast<int32_t*>(ws + at); };
  const Routes r = {i32(l.offsets),     i32(l.n_tiles), reinterpret_cast<int4*>(ws + l.tiles),
                    i32(l.tile_count),  i32(l.route_token), reinterpret_cast<float*>(ws + l.route_weight), i32(l.pick_route),
                    i32(l.chunk_counts)};
  float* Cf = reinterpret_cast<float*>(ws + l.cf);
  uint8_t* Cq = ws + l.cq;
  float* Cs = reinterpret_cast<float*>(ws + l.cs);
  float* Y = reinterpret_cast<float*>(ws + l.y);
  const int picks = a.T * a.k;
  hipError_t err;
  if (picks <= FEW_PICKS && a.I <= FEW_MAX_I) {
    const size_t tiles = max_tiles(picks, a.e_local, 16);
    const int w = stream_waves(w4_chunks(a.H));
    few_gemm1_kernel<<<(unsigned)(tiles * (a.I / 16)), 64 * w, w * 2 * 1024, stream>>>(a, Cf);
    if ((err = hipGetLastError()) != hipSuccess) return err;
    few_gemm2_kernel<<<a.H / 32, FEW_THREADS, 16 * a.I, stream>>>(a, Cf);
    return hipGetLastError();
  }
  const bool tile = experts_in_tiles(a);
  const int fr = a.T <= 16 ? 1 : 2;
  const TilePlan plan = {tile ? 0 : 16 * fr, a.I / BLK, a.H / BLK, (a.H / 16 + 15) / 16, a.I / BLK,
                         1.0f / (float)(device_cus() * TILE_WGS)};
  if (picks <= SORT_SMALL) {
    sort_small_kernel<<<2, SORT_THREADS, 0, stream>>>(a.ids, a.weights, picks, a.k, a.e_local, a.offset, plan, r);
  } else {
    const int chunk = sort_chunk(picks), chunks = (picks + chunk - 1) / chunk;
    sort_count_kernel<<<chunks, SORT_THREADS, 0, stream>>>(a.ids, picks, chunk, a.e_local, a.offset, r);
    if ((err = hipGetLastError()) != hipSuccess) return err;
    sort_place_kernel<<<chunks + 1, SORT_THREADS, 0, stream>>>(a.ids, a.weights, picks, chunk, chunks, a.k, a.e_local,
                                                               a.offset, plan, r);
  }
  if ((err = hipGetLastError()) != hipSuccess) return err;
  const size_t bound = max_tiles(picks, a.e_local, tile ? 2 * TILE_COLS : 16 * fr);
  // Workgroups: every tile's slices, or as many tiles' as fit, which then loop.
  auto grid_of = [&](int slices) {
    const size_t fit = MAX_GRID / slices > 0 ? MAX_GRID / slices : 1;
    return (unsigned)((bound < fit ? bound : fit) * slices);
  };
  if (tile) {
    by_grids(bound * (a.I / BLK), [&](unsigned grid, int base) {
      experts_gemm1_tile_kernel<<<grid, TILE_THREADS, 0, stream>>>(a, r, base, Cq, Cs);
    });
    if ((err = hipGetLastError()) != hipSuccess) return err;
    by_grids(bound * ((a.H / 16 + 15) / 16), [&](unsigned grid, int base) {
      experts_gemm2_tile_kernel<<<grid, TILE_THREADS, 0, stream>>>(a, r, base, Cq, Cs, Y);
    });
    if ((err = hipGetLastError()) != hipSuccess) return err;
    experts_combine_kernel<<<dim3(a.T, (a.H + 1023) / 1024), 256, 0, stream>>>(Y, r.pick_route, a.H, a.k, a.out);
    return hipGetLastError();
  }
  auto waves_of = [](int K) { return stream_waves(w4_chunks(K)); };
  {
    const int w = waves_of(a.H);
    const unsigned grid = grid_of(a.I / 16);
    if (fr == 1) experts_gemm1_kernel<1><<<grid, 64 * w, w * 2 * 1024, stream>>>(a, r, Cf);
    else experts_gemm1_kernel<2><<<grid, 64 * w, w * 4 * 1024, stream>>>(a, r, Cf);
    if ((err = hipGetLastError()) != hipSuccess) return err;
  }
  const size_t units = (size_t)picks * (a.I / BLK);
  requant_kernel<<<(unsigned)(units < 16 * 2048 ? (units + 15) / 16 : 2048), 256, 0, stream>>>(Cf, r.offsets + a.e_local,
                                                                                               a.I / BLK, Cq, Cs);
  if ((err = hipGetLastError()) != hipSuccess) return err;
  {
    const int w = waves_of(a.I);
    const unsigned grid = grid_of(a.H / 32);
    if (fr == 1) experts_gemm2_kernel<2, 1><<<grid, 64 * w, w * 2 * 1024, stream>>>(a, r, Cq, Cs, Y);
    else experts_gemm2_kernel<2, 2><<<grid, 64 * w, w * 4 * 1024, stream>>>(a, r, Cq, Cs, Y);
    if ((err = hipGetLastError()) != hipSuccess) return err;
  }
  experts_combine_kernel<<<dim3(a.T, (a.H + 1023) / 1024), 256, 0, stream>>>(Y, r.pick_route, a.H, a.k, a.out);
  return hipGetLastError();
}

}  // namespace moe
