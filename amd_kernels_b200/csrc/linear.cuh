// The MXFP8 matrix product y = act(x @ w^T + bias) + residual: what its kernels share. Formats, arguments, epilogue arithmetic.
#pragma once
#include "add_rmsnorm.cuh"
#include "tc_ptx.cuh"

namespace b200moe {

// Weights: first the codes, [row tile][K-tile] images of 128 weight rows x 128 K-elements, 16384 bytes of E4M3 as the 128-byte swizzle
// lays them in shared memory; behind them the scales, [row tile][K-tile] atoms of 512 bytes, so that those of several K-tiles are one
// copy. Rows and columns beyond the matrix are zero codes with scale byte 127. Gated weights (gate rows, then up rows) are interleaved in groups of 32,
// [gate 32 | up 32 | gate 32 | up 32], so that a tile holds 64 output columns with both halves.
constexpr int kLinearImageBytes = 128 * 128;
constexpr int kLinearTileBytes = kLinearImageBytes + kAtomBytes;

// Scales travel in groups of four K-tiles, ahead of the codes: two or three groups in shared memory, kSfSets in tensor memory. A copy, its
// waits and its commit then cost the issuing warps a quarter, and the MMAs never wait for a scale that came with its codes.
constexpr int kSfGroup = 4, kSfSets = 2;

// What the epilogue does with a sum p (or a gate g and an up u):
//   kLinear   max(p, floor) (ReLU: 0, none: -inf)
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
  const __nv_bfloat16* x;         // where the kernel quantises the rows itself: rows x_stride apart, in place of codes and scales
  const __nv_bfloat16* residual;  // rows residual_stride apart, or null
  __nv_bfloat16* out;             // rows out_stride apart; or null:
  uint8_t* out_codes;             // [m][n]
  uint8_t* out_scales;            // [m][n / 32]
  int64_t m, x_stride, residual_stride, out_stride;
  int k, n;  // n: output columns
  int tiles_n, tiles_k;
  LinearAct act;
};

// of[splits]: clusters of so many CTAs of the one-CTA kernel that are resident at once
struct LinearResident {
  int of[9];
};

// Two fp32 values an instruction (add, mul and fma of f32x2, each half rounded as the scalar one): the epilogues of wide products are
// bound by instructions, and by fetching them.
struct F2 {
  float x, y;
};
__device__ __forceinline__ uint64_t f2_bits(F2 v) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(v.x), "f"(v.y));
  return r;
}
__device__ __forceinline__ F2 f2_of(uint64_t r) {
  F2 v;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(v.x), "=f"(v.y) : "l"(r));
  return v;
}
__device__ __forceinline__ F2 f2_dup(float v) { return {v, v}; }
__device__ __forceinline__ F2 operator+(F2 a, F2 b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(f2_bits(a)), "l"(f2_bits(b)));
  return f2_of(r);
}
__device__ __forceinline__ F2 operator*(F2 a, F2 b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(f2_bits(a)), "l"(f2_bits(b)));
  return f2_of(r);
}
__device__ __forceinline__ F2 f2_fma(F2 a, F2 b, F2 c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(f2_bits(a)), "l"(f2_bits(b)), "l"(f2_bits(c)));
  return f2_of(r);
}
__device__ __forceinline__ F2 f2_exp2(F2 a) {  // 2^a, within 2 units in the last place
  F2 r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r.x) : "f"(a.x));
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r.y) : "f"(a.y));
  return r;
}
__device__ __forceinline__ F2 f2_rcp(F2 a) {  // 1 / a, within 1 unit in the last place; 0 for infinity
  F2 r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r.x) : "f"(a.x));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r.y) : "f"(a.y));
  return r;
}
__device__ __forceinline__ float min_nan(float a, float b) {  // NaN stays, as in the formulas
  float r;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

__device__ __forceinline__ float max3_abs(float a, float b, float c) {  // max(|a|, |b|, |c|); a NaN is skipped
  float r;
  asm("max.abs.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

constexpr float kLog2e = 1.4426950409f;
// The activations take N pairs a step at a time: a pair's own chain (an exponential, a reciprocal, GELU's polynomial) is far longer than what
// one instruction issues, and the compiler keeps the order that it is given.
#define FOR_PAIRS _Pragma("unroll") for (int k = 0; k < N; ++k)

template <int N>
__device__ __forceinline__ void act_linear(F2 (&p)[N], const LinearAct& a) {
  FOR_PAIRS p[k] = {max_nan(p[k].x, a.floor), max_nan(p[k].y, a.floor)};
}
// p *= sigmoid(v), w = -v log2(e)
template <int N>
__device__ __forceinline__ void times_sigmoid(F2 (&p)[N], F2 (&w)[N]) {
  FOR_PAIRS w[k] = f2_exp2(w[k]);
  FOR_PAIRS w[k] = w[k] + f2_dup(1.0f);
  FOR_PAIRS w[k] = f2_rcp(w[k]);
  FOR_PAIRS p[k] = p[k] * w[k];
}
template <int N>
__device__ __forceinline__ void act_sigmoid(F2 (&p)[N], const LinearAct& a) {
  F2 w[N];
  const F2 c1 = f2_dup(-kLog2e * a.c1);
  if (a.c3 == 0.0f) {
    FOR_PAIRS w[k] = p[k] * c1;
  } else {
    const F2 c3 = f2_dup(-kLog2e * a.c3);
    FOR_PAIRS w[k] = p[k] * p[k];
    FOR_PAIRS w[k] = f2_fma(w[k], c3, c1);
    FOR_PAIRS w[k] = p[k] * w[k];
  }
  times_sigmoid(p, w);
}
// p Phi(p) = max(p, 0) - |p| erfc(z) / 2, z = |p| / sqrt(2), and erfc(z) = exp(-z^2) t Q(t) with t = 1 / (1 + 0.427 z): Q of degree 7 is a
// fit of this file's (least squares, weighted until the largest relative error up to z = 8.5 is least: 6.7e-8, a step of fp32 is 1.2e-7),
// so that the negative tail keeps its relative precision. The coefficients carry the minus sign, the exponent (to base 2) the half. Measured, root
// mean square relative to the result: 1.4e-7 for p in -1.5 .. 0, 7e-8 in 0 .. 1.5. (A fit of degree 5, 2.9e-6, had 2.1e-6 and 9.7e-7 there, which
// moves codes of 8 bits over their borders, for 1.2 % of 2048 x 800 -> 5984: 28.2 / 28.6 us.)
template <int N>
__device__ __forceinline__ void act_gelu(F2 (&p)[N]) {
  F2 m[N], s[N], q[N];
  FOR_PAIRS m[k] = {fminf(fabsf(p[k].x), 64.0f), fminf(fabsf(p[k].y), 64.0f)};  // (erfc is 0 there; infinity times 0 is not)
  FOR_PAIRS s[k] = f2_fma(m[k], f2_dup(0.3019346f), f2_dup(1.0f));
  FOR_PAIRS s[k] = f2_rcp(s[k]);
  FOR_PAIRS q[k] = f2_fma(s[k], f2_dup(-0.0743070617f), f2_dup(0.32005927f));
  FOR_PAIRS q[k] = f2_fma(q[k], s[k], f2_dup(-0.411640257f));
  FOR_PAIRS q[k] = f2_fma(q[k], s[k], f2_dup(0.108598039f));
  FOR_PAIRS q[k] = f2_fma(q[k], s[k], f2_dup(-0.258320153f));
  FOR_PAIRS q[k] = f2_fma(q[k], s[k], f2_dup(-0.200422898f));
  FOR_PAIRS q[k] = f2_fma(q[k], s[k], f2_dup(-0.243175149f));
  FOR_PAIRS q[k] = f2_fma(q[k], s[k], f2_dup(-0.240791813f));
  FOR_PAIRS q[k] = q[k] * s[k];
  FOR_PAIRS s[k] = f2_fma(m[k] * m[k], f2_dup(-0.5f * kLog2e), f2_dup(-1.0f));
  FOR_PAIRS s[k] = f2_exp2(s[k]);
  FOR_PAIRS q[k] = q[k] * s[k];  // -erfc / 2
  FOR_PAIRS p[k] = f2_fma(m[k], q[k], F2{max_nan(p[k].x, 0.0f), max_nan(p[k].y, 0.0f)});
}
// g becomes min(g, top) sigmoid(c1 min(g, top)) (clamp(u) + beta)
template <int N>
__device__ __forceinline__ void act_gated(F2 (&g)[N], const F2 (&u)[N], const LinearAct& a) {
  F2 w[N];
  const F2 c1 = f2_dup(-kLog2e * a.c1);
  FOR_PAIRS g[k] = {min_nan(g[k].x, a.top), min_nan(g[k].y, a.top)};
  FOR_PAIRS w[k] = g[k] * c1;
  times_sigmoid(g, w);
  FOR_PAIRS g[k] = g[k] * (F2{max_nan(min_nan(u[k].x, a.top), -a.top), max_nan(min_nan(u[k].y, a.top), -a.top)} + f2_dup(a.beta));
}
template <int KIND, int N>
__device__ __forceinline__ void act_of(F2 (&p)[N], const LinearAct& a) {
  if (KIND == kLinear) act_linear(p, a);
  else if (KIND == kSigmoid) act_sigmoid(p, a);
  else act_gelu(p);
}
#undef FOR_PAIRS

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

// The row-major scales of the tokens: the 16 bytes of K-tiles kt .. kt + 3 (4 a K-tile) of ROWS rows, 32 apart, a lane. Asked for by load(),
// without a branch between the loads of one call, so that all of them are in flight together; put in order by tiles().
// `alignment`: rows begin at multiples of 16 bytes (K a multiple of 512), of 4 (of 128), or anywhere. Anywhere, a row's bytes are in five
// aligned words; those that reach over the ends of the array are not read, and the rows beside the ends are read by bytes.
struct RowScales {
  const uint8_t *base, *end;
  int64_t rows;
  int per_row, alignment;
  __device__ __forceinline__ RowScales(const uint8_t* scales, int64_t m, int k)
      : base(scales), end(scales + m * (k / 32)), rows(m), per_row(k / 32) {
    const uintptr_t at = reinterpret_cast<uintptr_t>(scales) | static_cast<uintptr_t>(per_row);
    alignment = (at & 15) == 0 ? 16 : (at & 3) == 0 ? 4 : 1;
  }
  // asks L2 for the line in which those bytes begin (before the launch in front has ended: L2 is where its stores go)
  template <int ROWS>
  __device__ __forceinline__ void prefetch(int64_t row, int kt) const {
#pragma unroll
    for (int i = 0; i < ROWS; ++i)
      if (row + 32 * i < rows) asm volatile("prefetch.global.L2 [%0];" ::"l"(base + (row + 32 * i) * per_row + kt * 4));
  }
  template <int ROWS>
  __device__ __forceinline__ void load(int64_t row, int kt, uint32_t (&w)[ROWS][5]) const {
    const uint8_t* p = base + row * per_row + kt * 4;
    const int64_t step = 32 * static_cast<int64_t>(per_row);
    if (alignment == 16 && (kt & 3) == 0) {  // (16 bytes divide the row)
#pragma unroll
      for (int i = 0; i < ROWS; ++i) {
        const uint4 v = row + 32 * i < rows ? __ldcg(reinterpret_cast<const uint4*>(p + i * step)) : make_uint4(0u, 0u, 0u, 0u);
        w[i][0] = v.x, w[i][1] = v.y, w[i][2] = v.z, w[i][3] = v.w;
      }
    } else if (alignment >= 4) {
#pragma unroll
      for (int i = 0; i < ROWS; ++i)
#pragma unroll
        for (int d = 0; d < 4; ++d)
          w[i][d] = row + 32 * i < rows && (kt + d) * 4 < per_row ? __ldcg(reinterpret_cast<const uint32_t*>(p + i * step) + d) : 0u;
    } else {
#pragma unroll
      for (int i = 0; i < ROWS; ++i) {
        const uint8_t* q = p + i * step - (reinterpret_cast<uintptr_t>(p + i * step) & 3);
#pragma unroll
        for (int d = 0; d < 5; ++d)
          w[i][d] = row + 32 * i < rows && q + 4 * d >= base && q + 4 * d + 4 <= end ? __ldcg(reinterpret_cast<const uint32_t*>(q) + d) : 0u;
      }
    }
  }
  // one row by bytes: the four words of K-tiles kt .. kt + 3
  __device__ __noinline__ uint4 by_bytes(int64_t row, int kt) const {
    uint32_t v[4] = {0u, 0u, 0u, 0u};
    for (int j = 0; j < 16 && kt * 4 + j < per_row; ++j) {
      const uint32_t b = static_cast<uint32_t>(__ldcg(base + row * per_row + kt * 4 + j)) << (8 * (j & 3));
      v[0] |= j < 4 ? b : 0u, v[1] |= j >= 4 && j < 8 ? b : 0u, v[2] |= j >= 8 && j < 12 ? b : 0u, v[3] |= j >= 12 ? b : 0u;
    }
    return make_uint4(v[0], v[1], v[2], v[3]);
  }
  // the loaded words -> w[i][d]: the four bytes of K-tile kt + d; 0 beyond the rows and the columns
  template <int ROWS>
  __device__ __forceinline__ void tiles(int64_t row, int kt, uint32_t (&w)[ROWS][5]) const {
    if (alignment >= 4) return;
    const int left = per_row - kt * 4;  // bytes of a row from K-tile kt on
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
      const int64_t r = row + 32 * i;
      const uint8_t* p = base + r * per_row + kt * 4;
      const int shift = 8 * static_cast<int>(reinterpret_cast<uintptr_t>(p) & 3);
#pragma unroll
      for (int d = 0; d < 4; ++d) {
        w[i][d] = __funnelshift_r(w[i][d], w[i][d + 1], shift);
        if (left < 4 * d + 4) w[i][d] &= left <= 4 * d ? 0u : 0xffffffffu >> (8 * (4 * d + 4 - left));  // the next row's bytes
      }
      if (r < rows && (p - base < 4 || end - p < 20)) {
        const uint4 v = by_bytes(r, kt);
        w[i][0] = v.x, w[i][1] = v.y, w[i][2] = v.z, w[i][3] = v.w;
      }
    }
  }
};

// 32 bytes, one sector, by one thread (32-byte aligned)
__device__ __forceinline__ void st_sector(void* p, const uint32_t (&w)[8]) {
  asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(p), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]), "r"(w[4]),
               "r"(w[5]), "r"(w[6]), "r"(w[7])
               : "memory");
}

// The code producer (warp 0) starts behind the scale producer's (warp 3) first requests: behind a full ring of codes of all SMs the scales
// took 5000 cycles to come.
__device__ __forceinline__ void scales_first_wait() { asm volatile("bar.sync 3, 64;" ::: "memory"); }
__device__ __forceinline__ void scales_first_arrive() { asm volatile("bar.arrive 3, 64;" ::: "memory"); }

// a tensor map into the cache that the copies read it from
__device__ __forceinline__ void prefetch_map(const CUtensorMap* map) {
  asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(map)) : "memory");
}
// a tile of codes into L2, through its tensor map
__device__ __forceinline__ void tma_prefetch_2d(const CUtensorMap* map, int x, int y) {
  asm volatile("cp.async.bulk.prefetch.tensor.2d.L2.global [%0, {%1, %2}];" ::"l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y) : "memory");
}

__device__ __forceinline__ void fence_proxy_async() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

}  // namespace b200moe
