// The MXFP8 matrix product y = act(x @ w^T + bias) + residual: what its kernels share. Formats, epilogue arithmetic, arguments.
#pragma once
#include "add_rmsnorm.cuh"

namespace b200moe {

// Weights: records of 128 weight rows x 128 K-elements, [row tile][K-tile]: 16384 bytes of E4M3 codes in the 128-byte-swizzled
// shared-memory image, then one scale atom. Rows and columns beyond the matrix are zeros. Gated weights (gate rows, then up rows) are
// interleaved in groups of 32, [gate 32 | up 32 | gate 32 | up 32], so that a tile holds 64 output columns with both halves.
constexpr int kLinearCodeBytes = 128 * 128;
constexpr int kLinearRecordBytes = kLinearCodeBytes + kAtomBytes;  // 132 rows of 128 bytes

struct LinearArgs {
  const uint8_t* tiles;
  const float* bias;         // [weight rows] or null
  const uint8_t* codes;      // [m][k]
  const uint8_t* scales;     // [m][k / 32]
  const __nv_bfloat16* residual;  // rows residual_stride apart, or null
  __nv_bfloat16* out;        // rows out_stride apart; or, for MXFP8 output, null:
  uint8_t* out_codes;        // [m][n]
  uint8_t* out_scales;       // [m][n / 32]
  int64_t m, residual_stride, out_stride;
  int k, n;                  // n: output columns
  int tiles_n, tiles_k;
  int act;
};

__device__ __forceinline__ bool linear_gated(int act) { return act >= B200MOE_ACT_SWIGLU; }

// p is multiplied by the logistic function of c * p
__device__ __forceinline__ float times_sigmoid(float p, float c) { return __fdividef(p, 1.0f + __expf(-c * p)); }

__device__ __forceinline__ float activate(float p, int act) {
  switch (act) {
    case B200MOE_ACT_RELU: return p < 0.0f ? 0.0f : p;  // (NaN stays)
    case B200MOE_ACT_SILU: return times_sigmoid(p, 1.0f);
    case B200MOE_ACT_GELU: return p * normcdff(p);
    case B200MOE_ACT_GELU_TANH:  // 0.5 p (1 + tanh(u)) = p / (1 + exp(-2 u)), u = sqrt(2 / pi) (p + 0.044715 p^3)
      return __fdividef(p, 1.0f + __expf(-1.5957691216f * (p + 0.044715f * p * p * p)));
  }
  return p;
}

__device__ __forceinline__ float activate_gated(float g, float u, int act) {
  return act == B200MOE_ACT_SWIGLU ? times_sigmoid(g, 1.0f) * u : swiglu_oai(g, u);
}

// E8M0 byte of an MXFP8 block, the shared expert's rule (ceil_pow2(amax / 448), at least 1); an infinite block keeps a finite scale
__device__ __forceinline__ int linear_scale(float amax) {
  const int e = mxfp8_scale(amax);
  return e > 254 ? 254 : e;
}

__device__ __forceinline__ uint32_t pack_e4m3x4(float a, float b, float c, float d) {
  return cvt_e4m3x2(a, b) | (cvt_e4m3x2(c, d) << 16);
}

}  // namespace b200moe
