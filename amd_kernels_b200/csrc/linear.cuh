// The MXFP8 matrix product y = act(x @ w^T + bias) + residual: what its kernels share. Formats, arguments, epilogue arithmetic.
#pragma once
#include "add_rmsnorm.cuh"
#include "tc_ptx.cuh"

namespace b200moe {

// Weights: first the codes, [row tile][K-tile] images of 128 weight rows x 128 K-elements, 16384 bytes of E4M3 as the 128-byte swizzle
// lays them in shared memory; behind them the scales, [row tile][K-tile] atoms of 512 bytes, so that those of several K-tiles are one
// copy. Rows and columns beyond the matrix are zeros. Gated weights (gate rows, then up rows) are interleaved in groups of 32,
// [gate 32 | up 32 | gate 32 | up 32], so that a tile holds 64 output columns with both halves.
constexpr int kLinearImageBytes = 128 * 128;
constexpr int kLinearTileBytes = kLinearImageBytes + kAtomBytes;

// Scales travel in groups of four K-tiles, ahead of the codes: two or three groups in shared memory, kSfSets in tensor memory. A copy, its
// waits and its commit then cost the issuing warps a quarter, and the MMAs never wait for a scale that came with its codes.
constexpr int kSfGroup = 4, kSfSets = 2;

// What the epilogue does with a sum p (or a gate g and an up u):
//   kLinear   p, or 0 where p < floor (ReLU: 0, none: -inf)
//   kSigmoid  p * sigmoid(c1 p + c3 p^3): SiLU, and GELU in its tanh form, 0.5 (1 + tanh(v)) = sigmoid(2 v)
//   kGelu     p * Phi(p)
//   kGated    min(g, top) * sigmoid(c1 min(g, top)) * (clamp(u, -top, top) + beta)
enum LinearKind { kLinear = 0, kSigmoid = 1, kGelu = 2, kGated = 3 };
struct LinearAct {
  int kind;
  float floor, c1, c3, top, beta;
};

struct LinearArgs {
  const uint8_t* tiles;           // images
  const uint8_t* atoms;           // scale atoms
  const float* bias;              // [weight rows] or null
  const uint8_t* codes;           // [m][k]
  const uint8_t* scales;          // [m][k / 32]
  const __nv_bfloat16* residual;  // rows residual_stride apart, or null
  __nv_bfloat16* out;             // rows out_stride apart; or null:
  uint8_t* out_codes;             // [m][n]
  uint8_t* out_scales;            // [m][n / 32]
  int64_t m, residual_stride, out_stride;
  int k, n;  // n: output columns
  int tiles_n, tiles_k;
  LinearAct act;
};

// NaN passes every clamp here (the comparison is false), as it does in the formulas
__device__ __forceinline__ float act_linear(float p, const LinearAct& a) { return p < a.floor ? 0.0f : p; }
__device__ __forceinline__ float act_sigmoid(float p, const LinearAct& a) {
  const float v = p * fmaf(a.c3, fminf(p * p, 1e30f), a.c1);  // (bounded: 0 * inf is NaN)
  return __fdividef(p, 1.0f + __expf(-v));
}
// Phi(p) = erfc(-p / sqrt(2)) / 2. erfc(z) = t exp(-z^2 + P(t)), t = 1 / (1 + z / 2), z >= 0: the Chebyshev fit of Numerical Recipes
// (erfcc), off by at most 1.2e-7 of its value everywhere, so that the negative tail keeps its relative precision; a third of the
// instructions of normcdff.
__device__ __forceinline__ float act_gelu(float p) {
  const float z = fabsf(p) * 0.70710678f, t = __fdividef(1.0f, fmaf(0.5f, z, 1.0f));
  float q = 0.17087277f;
  q = fmaf(q, t, -0.82215223f);
  q = fmaf(q, t, 1.48851587f);
  q = fmaf(q, t, -1.13520398f);
  q = fmaf(q, t, 0.27886807f);
  q = fmaf(q, t, -0.18628806f);
  q = fmaf(q, t, 0.09678418f);
  q = fmaf(q, t, 0.37409196f);
  q = fmaf(q, t, 1.00002368f);
  q = fmaf(q, t, -1.26551223f);
  const float half = 0.5f * t * __expf(fmaf(-z, z, q));  // erfc(z) / 2
  return p * (p < 0.0f ? half : 1.0f - half);
}
__device__ __forceinline__ float act_gated(float g, float u, const LinearAct& a) {
  g = g > a.top ? a.top : g;
  u = u > a.top ? a.top : u < -a.top ? -a.top : u;
  return g * __fdividef(1.0f, 1.0f + __expf(-a.c1 * g)) * (u + a.beta);
}
template <int KIND>
__device__ __forceinline__ float act_of(float p, const LinearAct& a) {
  return KIND == kLinear ? act_linear(p, a) : KIND == kSigmoid ? act_sigmoid(p, a) : act_gelu(p);
}

// E8M0 byte of an MXFP8 block, the shared expert's rule (ceil_pow2(amax / 448), at least 1); an infinite block keeps a finite scale
__device__ __forceinline__ int linear_scale(float amax) {
  const int e = mxfp8_scale(amax);
  return e > 254 ? 254 : e;
}
__device__ __forceinline__ uint32_t pack_e4m3x4(float a, float b, float c, float d) {
  return cvt_e4m3x2(a, b) | (cvt_e4m3x2(c, d) << 16);
}
__device__ __forceinline__ uint32_t pack_bf16x2(float a, float b) {
  const __nv_bfloat162 p = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&p);
}

// The row-major scales of the tokens. `alignment`: rows begin at multiples of 16 bytes (K a multiple of 512), of 4 (of 128), or anywhere.
struct RowScales {
  const uint8_t* base;
  int64_t rows;
  int per_row, alignment;
  __device__ __forceinline__ RowScales(const uint8_t* scales, int64_t m, int k) : base(scales), rows(m), per_row(k / 32) {
    const uintptr_t at = reinterpret_cast<uintptr_t>(scales) | static_cast<uintptr_t>(per_row);
    alignment = (at & 15) == 0 ? 16 : (at & 3) == 0 ? 4 : 1;
  }
  // The four bytes from the aligned address p on, those outside the array as zeros.
  __device__ __forceinline__ uint32_t word(const uint8_t* p) const {
    const uint8_t* end = base + rows * per_row;
    if (p >= base && p + 4 <= end) return __ldcg(reinterpret_cast<const uint32_t*>(p));
    uint32_t v = 0u;
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (p + j >= base && p + j < end) v |= static_cast<uint32_t>(__ldcg(p + j)) << (8 * j);
    return v;
  }
  // The bytes of K-tiles kt .. kt + 3 of a row, 4 a K-tile; 0 beyond the rows and the columns
  __device__ __forceinline__ uint4 at(int64_t row, int kt) const {
    if (row >= rows) return make_uint4(0u, 0u, 0u, 0u);
    const uint8_t* p = base + row * per_row + kt * 4;
    if (alignment == 16 && (kt & 3) == 0) return __ldcg(reinterpret_cast<const uint4*>(p));  // (16 bytes divide the row)
    uint32_t v[4] = {0u, 0u, 0u, 0u};
    const int left = per_row - kt * 4;  // bytes of the row from p on
    if (alignment >= 4) {
#pragma unroll
      for (int d = 0; d < 4; ++d)
        if (4 * d < left) v[d] = __ldcg(reinterpret_cast<const uint32_t*>(p) + d);
    } else {  // aligned words, shifted
      const int shift = static_cast<int>(reinterpret_cast<uintptr_t>(p) & 3);
      uint32_t w[5];
#pragma unroll
      for (int d = 0; d < 5; ++d) w[d] = 4 * d - shift < left ? word(p - shift + 4 * d) : 0u;
#pragma unroll
      for (int d = 0; d < 4; ++d) {
        v[d] = __funnelshift_r(w[d], w[d + 1], 8 * shift);
        if (left < 4 * d + 4) v[d] &= left <= 4 * d ? 0u : 0xffffffffu >> (8 * (4 * d + 4 - left));  // the next row's bytes
      }
    }
    return make_uint4(v[0], v[1], v[2], v[3]);
  }
};
__device__ __forceinline__ uint32_t word_of(const uint4 v, int d) { return d == 0 ? v.x : d == 1 ? v.y : d == 2 ? v.z : v.w; }

// 32 bytes, one sector, by one thread (32-byte aligned)
__device__ __forceinline__ void st_sector(void* p, const uint32_t (&w)[8]) {
  asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(p), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]), "r"(w[4]),
               "r"(w[5]), "r"(w[6]), "r"(w[7])
               : "memory");
}

__device__ __forceinline__ void fence_proxy_async() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

}  // namespace b200moe
