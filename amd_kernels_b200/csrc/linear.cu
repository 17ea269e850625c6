// The MXFP8 matrix product with bias, activation and residual in its epilogue: weight layout, row quantiser, entry point.
#include <math.h>

#include "linear.cuh"
#include "tc_host.cuh"

namespace b200moe {

// ------------------------------------------------------------------------------------------------ weight layout
// One CTA per (row of a tile, tile): 16-byte pieces of the source row into the swizzled images, its scales into the atoms.
__global__ void preshuffle_linear_kernel(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ scales, int64_t rows, int k,
                                         int tiles_k, int gated, uint8_t* __restrict__ out) {
  const int64_t t = blockIdx.x >> 7, tiles = static_cast<int64_t>(gridDim.x >> 7) * tiles_k;
  const int r = static_cast<int>(blockIdx.x & 127u);
  int64_t src = t * 128 + r;
  bool have = src < rows;
  if (gated) {
    const int g = r >> 5;
    const int64_t half = rows / 2, i = 64 * t + 32 * (g >> 1) + (r & 31);
    have = i < half;
    src = (g & 1) ? half + i : i;
  }
  uint8_t* image0 = out + t * tiles_k * kLinearImageBytes;
  uint8_t* atom0 = out + tiles * kLinearImageBytes + t * tiles_k * kAtomBytes;
  for (int j = threadIdx.x; j < tiles_k * 8; j += blockDim.x) {
    const int kt = j >> 3, c = j & 7;
    uint4 v = make_uint4(0u, 0u, 0u, 0u);
    if (have && j * 16 < k) v = *reinterpret_cast<const uint4*>(codes + src * k + j * 16);
    *reinterpret_cast<uint4*>(image0 + static_cast<int64_t>(kt) * kLinearImageBytes + r * 128 + ((c ^ (r & 7)) << 4)) = v;
  }
  for (int j = threadIdx.x; j < tiles_k * 4; j += blockDim.x)
    atom0[static_cast<int64_t>(j >> 2) * kAtomBytes + atom_offset(r, j & 3)] =
        have && j * 32 < k ? scales[src * (k / 32) + j] : static_cast<uint8_t>(127);
}

// ------------------------------------------------------------------------------------------------ row quantiser
// bf16 rows -> E4M3 codes and E8M0 scales, row-major. HBM bound: 2 bytes in, 33/32 out a value. blockDim = (threads of a row, rows of the
// CTA), up to V vectors of 8 a thread, all asked for at once; four lanes to a block of 32 values. (A thread for each vector of the
// whole array, its row found by a division, took 64 us for 16384 x 6144 where this takes 56.)
template <int V>
__global__ void __launch_bounds__(512) quant_mxfp8_kernel(const uint4* x, int64_t x_stride, int64_t rows, int vectors, uint2* codes,
                                                          uint8_t* scales) {
  pdl_enter(x);
  const int64_t row = static_cast<int64_t>(blockIdx.x) * blockDim.y + threadIdx.y;
  const int lane = threadIdx.x & 31, c0 = blockIdx.y * V * blockDim.x + threadIdx.x;  // (very wide rows are cut)
  const bool words = (vectors & 15) == 0 && (reinterpret_cast<uintptr_t>(scales) & 3) == 0;  // four scales of 16 lanes are a word
  uint4 raw[V];
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const int c = c0 + i * blockDim.x;
    raw[i] = row < rows && c < vectors ? __ldcg(x + row * x_stride + c) : make_uint4(0u, 0u, 0u, 0u);
  }
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const int c = c0 + i * blockDim.x;
    const bool in = row < rows && c < vectors;
    float v[8];
    unpack_bf16x8(raw[i], v);
    float amax = max3_abs(max3_abs(v[0], v[1], v[2]), max3_abs(v[3], v[4], v[5]), max3_abs(v[6], v[7], 0.0f));
    amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
    amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
    const int e = linear_scale(amax);
    const float inv = e8m0_value(static_cast<uint32_t>(254 - e));
    uint32_t sc = static_cast<uint32_t>(e);
    if (words) {
      sc |= __shfl_down_sync(0xffffffffu, sc, 4) << 8;
      sc |= __shfl_down_sync(0xffffffffu, sc, 8) << 16;
    }
    if (!in) continue;
    codes[row * vectors + c] = make_uint2(pack_e4m3x4(v[0] * inv, v[1] * inv, v[2] * inv, v[3] * inv),
                                          pack_e4m3x4(v[4] * inv, v[5] * inv, v[6] * inv, v[7] * inv));
    uint8_t* s = scales + row * (vectors >> 2) + (c >> 2);
    if (words && (lane & 15) == 0) *reinterpret_cast<uint32_t*>(s) = sc;
    if (!words && (lane & 3) == 0) *s = static_cast<uint8_t>(e);
  }
}

template <int V>
static int launch_quant(const uint4* x, int64_t x_stride, int64_t rows, int vectors, uint2* codes, uint8_t* scales, cudaStream_t stream) {
  const int wide = vectors < V * 512 ? vectors : V * 512;
  const int threads = ((wide + V - 1) / V + 31) / 32 * 32, rows_per_cta = threads >= 128 ? 1 : 256 / threads;
  const int64_t grid = (rows + rows_per_cta - 1) / rows_per_cta;
  B200MOE_LAUNCH(quant_mxfp8_kernel<V>, dim3(static_cast<unsigned>(grid), (vectors + V * threads - 1) / (V * threads)),
                 dim3(threads, rows_per_cta), 0, stream, x, x_stride, rows, vectors, codes, scales);
  return 0;
}

// ------------------------------------------------------------------------------------------------ the call
int linear_tc(const LinearArgs& a, int bm, int splits, int32_t* status, cudaStream_t stream);  // linear_tc.cu
LinearResident linear_tc_resident(int bm);
int linear_pair(const LinearArgs& a, int32_t* status, cudaStream_t stream);  // linear_pair.cu
int linear_pair_resident(const LinearArgs& a);
int set_wait_limit_linear_tc(unsigned long long ns);
int set_wait_limit_linear_pair(unsigned long long ns);

static LinearAct act_args(int activation) {
  LinearAct a = {kLinear, -INFINITY, 1.0f, 0.0f, INFINITY, 0.0f};
  switch (activation) {
    case B200MOE_ACT_RELU: a.floor = 0.0f; break;
    case B200MOE_ACT_SILU: a.kind = kSigmoid; break;
    case B200MOE_ACT_GELU: a.kind = kGelu; break;
    case B200MOE_ACT_GELU_TANH:  // 2 sqrt(2 / pi) (p + 0.044715 p^3)
      a.kind = kSigmoid, a.c1 = 1.5957691216f, a.c3 = 1.5957691216f * 0.044715f;
      break;
    case B200MOE_ACT_SWIGLU: a.kind = kGated; break;
    case B200MOE_ACT_SWIGLU_OAI: a.kind = kGated, a.c1 = 1.702f, a.top = 7.0f, a.beta = 1.0f; break;
  }
  return a;
}

static int64_t linear_row_tiles(int64_t rows) { return (rows + 127) / 128; }  // gated: 64 output columns, 128 rows, as well
static int64_t linear_k_tiles(int64_t k) { return (k + 127) / 128; }

static bool linear_dims(int64_t rows, int64_t k, int gated) {
  if (rows < 8 || k < 32 || k % 32 || rows % (gated ? 64 : 8) || rows > B200MOE_LINEAR_MAX_DIM || k > B200MOE_LINEAR_MAX_DIM) return false;
  // the images seen as rows of 128 bytes are counted in 32 bits (274 GB)
  return linear_row_tiles(rows) * linear_k_tiles(k) <= INT32_MAX / 128;
}

int set_wait_limit_linear(unsigned long long ns) {
  const int r = set_wait_limit_linear_tc(ns);
  return r ? r : set_wait_limit_linear_pair(ns);
}

// CTAs along K for `units` (weight tile, token block). All clusters have to be resident at once: a second round of them costs more than any
// split gives (6144 -> 6144, one row, 10.2 us with 4, 15.8 with 6). Of 4, 6 and 8 the one whose longest part has the fewest groups of
// four K-tiles; of equals the smallest, the largest up to 8 units: one row 6144 -> 2560 with 4 / 6 / 8 8.1 / 7.1 / 7.3 (3 / 2 / 2 groups),
// 4096 -> 1024 6.1 / 5.7 / 5.1 (2 / 2 / 1), 6144 -> 1024 7.3 / 6.3 / 5.8, 1536 -> 2048 4.6 each (1); 64 rows 6144 -> 5120 13.0 / 12.0.
// With more than 32 rows a block 6 and 8 only where their parts are whole groups: 100 rows 8192 -> 2048 11.9 / 12.6. (Where 4 put a CTA on
// each SM, 6 can lose: 16 rows 6144 -> 4096 8.9 / 9.3; one row 8.5 / 8.3.) Else 2 or 1. 0: no one round.
static int splits_for(const LinearArgs& a, int bm, int64_t units) {
  const LinearResident resident = linear_tc_resident(bm);
  int best = 0, best_groups = 0;
  for (int splits : {4, 6, 8, 2, 1}) {
    if (units <= 8 && splits >= 4) splits = 12 - splits;
    if (splits > a.tiles_k || (splits < 4 && best) || units > resident.of[splits]) continue;
    if (splits > 4 && bm > 32 && a.tiles_k % (splits * kSfGroup)) continue;
    const int groups = ((a.tiles_k + splits - 1) / splits + kSfGroup - 1) / kSfGroup;
    if (!best || groups < best_groups) best = splits, best_groups = groups;
  }
  return best;
}

// The kernel, its token block and its split of K. Measured, us, 6144 -> 6144 (4096; 12288) unless said otherwise:
//   up to 128 rows the smallest block that holds them, so that the weights stream once; but two blocks of half the rows where these
//   still split K by 4 (33 to 64 rows: 10.6 / 11.2 at 4096; 13.7 / 13.1 at 6144 with a split of 2) or by 2 (65 to 128 rows: 12.4 / 14.8 at
//   4096, 15.6 / 16.6 at 6144; 23.9 / 22.0 at 12288 without a split).
//   More rows: blocks of 128 on one CTA while they split K by 2 in one round, else CTA pairs: 256 rows 20.2 / 23.9, 384 20.8 / 24.1, 512
//   30.6 / 24.4; 1024 rows 6144 -> 2048 19.6 / 22.7, 1536 29.9 / 24.0. Without a split too where they need one round and the pairs two
//   (384 rows at 12288: 33.3 / 39.7).
static int dispatch_linear(const LinearArgs& a, int32_t* status, cudaStream_t stream) {
  const int64_t blocks = (a.m + 127) / 128;
  int bm = a.m <= 16 ? 16 : a.m <= 32 ? 32 : a.m <= 64 ? 64 : 128;
  int splits = splits_for(a, bm, blocks * a.tiles_n);
  if (blocks == 1 && bm >= 64) {
    const int half = splits_for(a, bm / 2, 2 * static_cast<int64_t>(a.tiles_n));
    if (half >= (bm == 64 ? 4 : 2) && 2 * half >= splits) bm /= 2, splits = half;
  }
  if (blocks > 1) {  // (no pair resident: the one-CTA kernel, which needs no cluster without a split, takes any size)
    const int64_t pairs = (a.m + 255) / 256 * ((a.tiles_n + 1) / 2);
    const int resident = linear_pair_resident(a);
    if (resident > 0 && (splits == 0 || (splits == 1 && pairs <= resident))) return linear_pair(a, status, stream);
  }
  return linear_tc(a, bm, splits ? splits : 1, status, stream);
}

}  // namespace b200moe

extern "C" size_t b200moe_linear_weight_bytes(int64_t rows, int64_t k, int gated) {
  using namespace b200moe;
  if (!linear_dims(rows, k, gated)) return 0;
  return static_cast<size_t>(linear_row_tiles(rows)) * linear_k_tiles(k) * kLinearTileBytes;
}

extern "C" int b200moe_preshuffle_linear(const uint8_t* codes, const uint8_t* scales, int64_t rows, int64_t k, int gated,
                                         uint8_t* tiles, void* stream) {
  using namespace b200moe;
  if (!codes || !scales || !tiles || !linear_dims(rows, k, gated)) return B200MOE_E_ARG;
  if (misaligned(codes, 16) || misaligned(tiles, 128)) return B200MOE_E_ALIGN;
  B200MOE_LAUNCH_PLAIN(preshuffle_linear_kernel, dim3(static_cast<unsigned>(linear_row_tiles(rows) * 128)), 128, 0,
                       static_cast<cudaStream_t>(stream), codes, scales, rows, static_cast<int>(k),
                       static_cast<int>(linear_k_tiles(k)), gated, tiles);
  return 0;
}

extern "C" int b200moe_quant_mxfp8(const void* x_bf16, int64_t x_stride, int64_t rows, int64_t k, uint8_t* codes8, uint8_t* scales8,
                                   void* stream) {
  using namespace b200moe;
  if (rows < 0 || rows > B200MOE_LINEAR_MAX_ROWS || k < 32 || k % 32 || k > B200MOE_LINEAR_MAX_DIM) return B200MOE_E_ARG;
  if (rows == 0) return 0;
  if (!x_bf16 || !codes8 || !scales8) return B200MOE_E_ARG;
  if (rows > 1 && x_stride < k && x_stride != 0) return B200MOE_E_ARG;
  if (misaligned(x_bf16, 16) || misaligned(codes8, 8) || (rows > 1 && (x_stride & 7))) return B200MOE_E_ALIGN;
  const RowSpan x = {x_bf16, rows, 2 * k, rows > 1 ? 2 * x_stride : 2 * k}, codes = {codes8, rows, k, k}, scales = {scales8, rows, k / 32, k / 32};
  if (rows_overlap(x, codes) || rows_overlap(x, scales) || rows_overlap(codes, scales)) return B200MOE_E_ARG;
  const int v = static_cast<int>(k / 8);
  return (v <= 1024 ? launch_quant<3> : launch_quant<8>)(static_cast<const uint4*>(x_bf16), x_stride / 8, rows, v,
                                                         reinterpret_cast<uint2*>(codes8), scales8, static_cast<cudaStream_t>(stream));
}

namespace b200moe {
// Checks a call and fills the kernels' arguments; a.m is 0 where there is nothing to do.
static int linear_args(LinearArgs& a, const b200moe_linear_call* call, const int32_t* status) {
  a.m = 0;
  if (!call) return B200MOE_E_ARG;
  const b200moe_linear_call& c = *call;
  const b200moe_linear_weights* w = &c.w;
  const int64_t m = c.m;
  if (m < 0 || m > B200MOE_LINEAR_MAX_ROWS || !linear_dims(w->rows, w->k, w->gated)) return B200MOE_E_ARG;
  if (c.activation < B200MOE_ACT_NONE || c.activation > B200MOE_ACT_SWIGLU_OAI) return B200MOE_E_ARG;
  if ((w->gated != 0) != (c.activation >= B200MOE_ACT_SWIGLU)) return B200MOE_E_ARG;
  if (m == 0) return 0;
  const bool inside = c.x && m <= B200MOE_LINEAR_ROWS_INSIDE;
  if (!w->tiles || !status || (!inside && (!c.codes8 || !c.scales8))) return B200MOE_E_ARG;
  if ((c.out != nullptr) == (c.out_codes8 != nullptr) || (c.out_codes8 != nullptr) != (c.out_scales8 != nullptr)) return B200MOE_E_ARG;
  const int64_t n = w->gated ? w->rows / 2 : w->rows;
  if (c.out_codes8 && n % 32) return B200MOE_E_ARG;
  if (c.x && m > 1 && c.x_stride < w->k && c.x_stride != 0) return B200MOE_E_ARG;
  if (m > 1 && ((c.out && c.out_stride < n) || (c.residual && c.residual_stride < n))) return B200MOE_E_ARG;
  const auto bad_rows = [m](const void* p, int64_t stride) { return misaligned(p, 16) || (p && m > 1 && (stride & 7)); };
  if (misaligned(w->tiles, 128) || misaligned(w->bias, 16) || bad_rows(c.x, c.x_stride) || misaligned(c.codes8, 16) || misaligned(c.out_codes8, 16) ||
      bad_rows(c.out, c.out_stride) || bad_rows(c.residual, c.residual_stride))
    return B200MOE_E_ALIGN;
  // the rows of out may be those of the residual (a thread stores where it has loaded); any other overlap with an input is refused
  const int64_t k = w->k, weight_bytes = linear_row_tiles(w->rows) * linear_k_tiles(k) * kLinearTileBytes;
  const auto bf16_rows = [m](const void* p, int64_t width, int64_t stride) { return RowSpan{p, m, 2 * width, m > 1 ? 2 * stride : 2 * width}; };
  const RowSpan outs[] = {bf16_rows(c.out, n, c.out_stride), {c.out_codes8, m, n, n}, {c.out_scales8, m, n / 32, n / 32}};
  const RowSpan residual = bf16_rows(c.residual, n, c.residual_stride);
  const RowSpan ins[] = {bf16_rows(c.x, k, c.x_stride), {inside ? nullptr : c.codes8, m, k, k}, {inside ? nullptr : c.scales8, m, k / 32, k / 32},
                         {w->tiles, 1, weight_bytes, weight_bytes}, {w->bias, 1, 4 * w->rows, 4 * w->rows}};
  const bool in_place = c.out && c.out == c.residual && (m == 1 || c.out_stride == c.residual_stride);
  for (const RowSpan& o : outs) {
    for (const RowSpan& i : ins)
      if (rows_overlap(o, i)) return B200MOE_E_ARG;
    if (!in_place && rows_overlap(o, residual)) return B200MOE_E_ARG;
  }
  if (rows_overlap(outs[1], outs[2])) return B200MOE_E_ARG;
  if (c.x && !inside) {  // the quantiser in front writes these two (and compares them with x): nothing else that the product reads
    for (const RowSpan& scratch : {ins[1], ins[2]})
      if (rows_overlap(scratch, residual) || rows_overlap(scratch, ins[3]) || rows_overlap(scratch, ins[4])) return B200MOE_E_ARG;
  }
  a.tiles = w->tiles;
  a.bias = w->bias;
  a.x = inside ? static_cast<const __nv_bfloat16*>(c.x) : nullptr;
  a.x_stride = c.x_stride;
  a.codes = c.codes8;
  a.scales = c.scales8;
  a.residual = static_cast<const __nv_bfloat16*>(c.residual);
  a.out = static_cast<__nv_bfloat16*>(c.out);
  a.out_codes = c.out_codes8;
  a.out_scales = c.out_scales8;
  a.m = m;
  a.residual_stride = c.residual_stride;
  a.out_stride = c.out_stride;
  a.k = static_cast<int>(w->k);
  a.n = static_cast<int>(n);
  a.tiles_n = static_cast<int>(linear_row_tiles(w->rows));
  a.tiles_k = static_cast<int>(linear_k_tiles(w->k));
  a.atoms = w->tiles + static_cast<int64_t>(a.tiles_n) * a.tiles_k * kLinearImageBytes;
  a.act = act_args(c.activation);
  return 0;
}
}  // namespace b200moe

extern "C" int b200moe_linear(const b200moe_linear_call* call, int32_t* status, void* stream) {
  using namespace b200moe;
  LinearArgs a;
  int r = linear_args(a, call, status);
  if (r || a.m == 0) return r;
  if (call->x && !a.x && (r = b200moe_quant_mxfp8(call->x, call->x_stride, call->m, call->w.k, call->codes8, call->scales8, stream))) return r;
  return dispatch_linear(a, status, static_cast<cudaStream_t>(stream));
}
