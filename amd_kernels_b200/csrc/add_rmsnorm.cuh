// What the fused tail (tail.cu) and the norm without slots (add_rmsnorm.cu) share: bf16 vectors and the norm's MXFP8 scale.
#pragma once
#include "common.cuh"

namespace b200moe {

__device__ __forceinline__ void unpack_bf16x8(const uint4 v, float (&f)[8]) {
  const uint32_t r[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    f[2 * j] = __uint_as_float(r[j] << 16);
    f[2 * j + 1] = __uint_as_float(r[j] & 0xffff0000u);
  }
}

__device__ __forceinline__ uint4 pack_bf16x8(const float (&f)[8]) {
  uint32_t o[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const __nv_bfloat162 p = __floats2bfloat162_rn(f[2 * j], f[2 * j + 1]);
    o[j] = *reinterpret_cast<const uint32_t*>(&p);
  }
  return make_uint4(o[0], o[1], o[2], o[3]);
}

// clamp(ceil(log2(a / 448)) + 127, 0, 254) for a >= 2^-126 (a may be +inf): the division rounded to fp32, then the
// exact ceiling of its base-2 logarithm read from the bits (subnormal quotients included).
__device__ __forceinline__ int tail_mxfp8_scale(float a) {
  const uint32_t u = __float_as_uint(__fdiv_rn(a, 448.0f));
  const int ef = static_cast<int>((u >> 23) & 255u);
  const uint32_t m = u & 0x7fffffu;
  int sb = ef ? ef + (m != 0u) : (m > 0x400000u ? 1 : 0);
  return sb > 254 ? 254 : sb;
}

}  // namespace b200moe
