// Residual addition -> RMS norm -> MXFP8 and / or bf16 rows, any row width: what stands in front of the MoE layer (behind the attention's
// output projection, or at a model's first layer) where tail.cu, which does the same behind a slot sum, has no slots to read.
//
// Per row of h columns:
//   s   = fp32(x) + fp32(residual)   (x alone without a residual);  residual_out = bf16(s)
//   y   = (s * rstd) * (weight + offset),  rstd = 1 / sqrt(sum(s^2) / h + eps)          (the norm reads the fp32 s)
//   out = bf16(y)                                                                       (optional)
//   per 32 columns of y: a = max(max|y|, 2^-126), scale byte = clamp(ceil(log2(a / 448)) + 127, 0, 254),
//   code = e4m3(y * 2^(127 - byte)), round to nearest even, saturating                  (optional)
// One pass: a row stays in registers between its sum of squares and its outputs. Every thread adds its own squares in rising column
// order, then a warp tree, then the warp sums in order: the bits of a row depend on its width alone, never on the other rows.
//
// Bound: HBM. 16384 x 6144 with a residual and all outputs, 909 MB, takes 145 us (0.96 of the copy rate); one row 2.6 us, what a launch and two
// trips to memory take. Wide rows keep fewer bytes in flight an SM (16384 columns: one CTA of 512 threads with 74 registers; above, the weights
// come behind the sum): 4096 x 8192 48 us (0.96 of the copy rate), 4096 x 16384 123 (0.75), 2048 x 32768 145 (0.64); one row of 32768 8.2.
#include "add_rmsnorm.cuh"
#include "tc_host.cuh"

namespace b200moe {

struct NormArgs {
  const uint4* x;         // rows x_stride vectors of 8 bf16 apart
  const uint4* residual;  // or null
  const uint4* weight;    // [h]
  uint4* residual_out;
  uint4* normed;    // or null
  uint2* codes8;    // [rows][h] or null
  uint8_t* scales8;
  int64_t x_stride, residual_stride, residual_out_stride, normed_stride, rows;
  int vectors;  // h / 8
  float h, offset, eps;
};

// blockDim = (threads of a row, a whole number of warps; rows of the CTA); a thread holds up to V vectors of its row
template <int V>
__global__ void __launch_bounds__(512) add_rmsnorm_kernel(const NormArgs args) {
  pdl_launch_dependents();
  pdl_wait();
  NormArgs a = args;
  launder(a.x);
  launder(a.residual);
  launder(a.weight);
  __shared__ float warp_sum[32];
  const int lane = threadIdx.x & 31, warps = blockDim.x >> 5;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * blockDim.y + threadIdx.y;
  const bool have = row < a.rows;
  float s[V][8];
  float ss = 0.0f;
  // All of a thread's loads are in flight together, the weights among them while the registers allow it: asked for behind the sum, they
  // cost 0.5 us of 3 for one row and 4 % of 16384 x 6144.
  constexpr bool kEarly = V <= 4;
  uint4 raw[V], res[V], wraw[kEarly ? V : 1];
  const uint4 zero = make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const int c = i * blockDim.x + threadIdx.x;
    const bool in = have && c < a.vectors;
    raw[i] = in ? __ldcg(a.x + row * a.x_stride + c) : zero;
    res[i] = in && a.residual != nullptr ? __ldcg(a.residual + row * a.residual_stride + c) : zero;
    if (kEarly) wraw[kEarly ? i : 0] = in ? __ldcg(a.weight + c) : zero;
  }
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const int c = i * blockDim.x + threadIdx.x;
    unpack_bf16x8(raw[i], s[i]);
    if (a.residual != nullptr) add_bf16x8(s[i], res[i]);
#pragma unroll
    for (int j = 0; j < 8; ++j) ss = fmaf(s[i][j], s[i][j], ss);
    if (a.residual_out != nullptr && have && c < a.vectors) a.residual_out[row * a.residual_out_stride + c] = pack_bf16x8(s[i]);
  }
#pragma unroll
  for (int off = 16; off; off >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, off);
  if (warps > 1) {
    if (lane == 0) warp_sum[threadIdx.y * warps + (threadIdx.x >> 5)] = ss;
    __syncthreads();
    ss = 0.0f;
    for (int w = 0; w < warps; ++w) ss += warp_sum[threadIdx.y * warps + w];
  }
  const float rstd = __frcp_rn(__fsqrt_rn(__fdiv_rn(ss, a.h) + a.eps));
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const int c = i * blockDim.x + threadIdx.x;
    const bool in = have && c < a.vectors;
    float wv[8], y[8];
    unpack_bf16x8(kEarly ? wraw[kEarly ? i : 0] : in ? __ldcg(a.weight + c) : zero, wv);
    float amax = 0.0f;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      y[j] = (s[i][j] * rstd) * (wv[j] + a.offset);
      amax = fmaxf(amax, fabsf(y[j]));  // fmaxf skips a NaN operand
    }
    if (a.normed != nullptr && in) a.normed[row * a.normed_stride + c] = pack_bf16x8(y);
    if (a.codes8 != nullptr) {  // the four lanes of a 32-column block are all inside the row or all outside (h % 32 == 0)
      amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
      amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
      const int sb = tail_mxfp8_scale(fmaxf(amax, 1.17549435e-38f));
      const float inv = e8m0_value(static_cast<uint32_t>(254 - sb));  // 2^(127 - sb)
      if (in) {
        a.codes8[row * a.vectors + c] = make_uint2(cvt_e4m3x2(y[0] * inv, y[1] * inv) | (cvt_e4m3x2(y[2] * inv, y[3] * inv) << 16),
                                                   cvt_e4m3x2(y[4] * inv, y[5] * inv) | (cvt_e4m3x2(y[6] * inv, y[7] * inv) << 16));
        if ((lane & 3) == 0) a.scales8[row * (a.vectors >> 2) + (c >> 2)] = static_cast<uint8_t>(sb);
      }
    }
  }
}

template <int V>
static int launch_norm(const NormArgs& a, int threads, int rows_per_cta, cudaStream_t stream) {
  const int64_t grid = (a.rows + rows_per_cta - 1) / rows_per_cta;
  if (grid > 0x7fffffff) return B200MOE_E_ARG;
  B200MOE_LAUNCH(add_rmsnorm_kernel<V>, dim3(static_cast<unsigned>(grid)), dim3(threads, rows_per_cta), 0, stream, a);
  return 0;
}

}  // namespace b200moe

extern "C" int b200moe_add_rmsnorm_quant(const b200moe_norm_call* call, void* stream) {
  using namespace b200moe;
  if (!call) return B200MOE_E_ARG;
  const b200moe_norm_call& c = *call;
  const int64_t rows = c.rows, h = c.h;
  if (rows < 0 || h < 32 || h > B200MOE_NORM_MAX_H || h % 32) return B200MOE_E_ARG;
  if (rows == 0) return 0;
  if (!c.x || !c.weight) return B200MOE_E_ARG;
  if ((c.codes8 != nullptr) != (c.scales8 != nullptr) || (c.residual_out && !c.residual)) return B200MOE_E_ARG;
  if (!c.residual_out && !c.normed && !c.codes8) return B200MOE_E_ARG;
  struct Rows { const void* p; int64_t stride, width; int size; bool out; };
  const Rows all[] = {{c.x, c.x_stride, h, 2, false},
                      {c.residual, c.residual_stride, h, 2, false},
                      {c.residual_out, c.residual_out_stride, h, 2, true},
                      {c.normed, c.normed_stride, h, 2, true},
                      {c.codes8, h, h, 1, true},
                      {c.scales8, h / 32, h / 32, 1, true},
                      {c.weight, h, h, 2, false}};
  constexpr int kAll = sizeof(all) / sizeof(all[0]);
  for (int i = 0; i < kAll; ++i) {
    const Rows& r = all[i];
    if (!r.p) continue;
    if (rows > 1 && (r.stride < r.width && !(i == 1 && r.stride == 0))) return B200MOE_E_ARG;  // (a residual that all rows share)
    if (i != 5 && (misaligned(r.p, i == 4 ? 8 : 16) || (r.size == 2 && rows > 1 && (r.stride & 7)))) return B200MOE_E_ALIGN;
  }
  // an output may be an input with the same rows (a thread stores where it has loaded); any other overlap is refused
  for (int i = 0; i < kAll; ++i) {
    if (!all[i].p || !all[i].out) continue;
    for (int j = 0; j < kAll; ++j) {
      if (!all[j].p || j == i || (all[j].out && j < i)) continue;
      const bool same = j < 2 && all[i].p == all[j].p && all[i].size == 2 && (rows <= 1 || all[i].stride == all[j].stride);
      const auto span = [&](int k) {
        const Rows& r = all[k];
        return RowSpan{r.p, k == 6 ? 1 : rows, r.width * r.size, rows > 1 ? r.stride * r.size : r.width * r.size};
      };
      if (!same && rows_overlap(span(i), span(j))) return B200MOE_E_ARG;
    }
  }
  NormArgs a;
  a.x = static_cast<const uint4*>(c.x);
  a.residual = static_cast<const uint4*>(c.residual);
  a.weight = static_cast<const uint4*>(c.weight);
  a.residual_out = static_cast<uint4*>(c.residual_out);
  a.normed = static_cast<uint4*>(c.normed);
  a.codes8 = reinterpret_cast<uint2*>(c.codes8);
  a.scales8 = c.scales8;
  a.x_stride = c.x_stride / 8;
  a.residual_stride = c.residual_stride / 8;
  a.residual_out_stride = c.residual_out_stride / 8;
  a.normed_stride = c.normed_stride / 8;
  a.rows = rows;
  a.vectors = static_cast<int>(h / 8);
  a.h = static_cast<float>(h);
  a.offset = c.weight_offset;
  a.eps = c.eps;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const int v = a.vectors;
  const auto threads = [v](int per_thread) { return ((v + per_thread - 1) / per_thread + 31) / 32 * 32; };
  if (v <= 256) return launch_norm<1>(a, threads(1), v <= 32 ? 8 : v <= 64 ? 4 : v <= 128 ? 2 : 1, st);
  if (v <= 512) return launch_norm<2>(a, threads(2), 1, st);
  if (v <= 768) return launch_norm<3>(a, threads(3), 1, st);
  if (v <= 2048) return launch_norm<4>(a, threads(4), 1, st);
  return launch_norm<8>(a, threads(8), 1, st);
}
