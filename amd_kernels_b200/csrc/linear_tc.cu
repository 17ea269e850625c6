// The MXFP8 product for few rows: tcgen05.mma kind::mxf8f6f4 block-scaled with the weight tile as the 128-row M operand and a block of
// BM token rows as N, so that one pass over the weights serves the whole block.
//
// What bounds it: the weight stream (HBM). One CTA = (weight tile, token block, part of K). K is split over the CTAs of a cluster until
// there are enough of them to keep every SM loading; each adds its part in tensor memory, writes it to its shared memory, and after a cluster barrier
// the CTAs share out the block's rows: the parts of a row are added in the order of K through distributed shared memory, then
// bias, activation, residual and the only rounding. No workspace, no atomics, one launch, sums in a fixed order.
//
//   warp 0     code producer: the weight image (one bulk copy of consecutive HBM bytes) and the token rows (TMA)
//   warp 1     tensor memory; issues the MMAs, the whole warp around one elected lane
//   warp 2     scales: shared memory -> tensor memory
//   warp 3     scale producer: the weights' atoms (bulk copy); the tokens' from row-major global memory through registers
//   warps 4-7  the sum out of tensor memory; all warps take part in what follows
#include "linear.cuh"
#include "tc_pair.cuh"

namespace b200moe {

template <int BM>
struct LinearCfg {
  static constexpr int kAtoms = BM > 128 ? 2 : 1;                            // token scale atoms of a K-tile
  static constexpr int kTokOff = kLinearImageBytes;                          // token rows behind the weight image
  static constexpr int kStageBytes = kTokOff + BM * 128;
  static constexpr int kCtasPerSm = BM > 128 ? 1 : 2;                        // two: one's start and end under the other's stream
  static constexpr int kStages = BM > 128 ? 4 : BM > 64 ? 3 : BM > 32 ? 4 : 5;
  static constexpr int kSfSlots = BM == 32 ? 2 : 3;                          // groups of scales in shared memory
  static constexpr int kSfOff = kStages * kStageBytes;
  static constexpr int kSfTileBytes = (1 + kAtoms) * kAtomBytes;             // a K-tile's scales in a slot: see below
  static constexpr int kSfSlotBytes = kSfGroup * kSfTileBytes;               // weight atoms of the group, then token atoms by K-tile
  static constexpr int kSumRow = 132;                                        // floats of a token's 128 columns in the parts (alias the ring)
  static constexpr int kSmemBytes = kSfOff + kSfSlots * kSfSlotBytes + 1024;
  static constexpr int kSfCols = kAtoms > 1 ? 16 : 8;                        // tensor memory columns of a K-tile's scales: weights, tokens
  static constexpr int kColsUsed = BM + kSfSets * kSfGroup * kSfCols;
  static constexpr int kTmemCols = kColsUsed <= 64 ? 64 : kColsUsed <= 128 ? 128 : kColsUsed <= 256 ? 256 : 512;
  static_assert(BM * kSumRow * 4 <= kSfOff, "the parts fit the ring");
  static_assert(kSmemBytes <= 227 * 1024 / kCtasPerSm - 1024 && kTmemCols * kCtasPerSm <= 512, "shared and tensor memory");
};

__device__ __forceinline__ float4 ld_cluster_f4(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0,%1,%2,%3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ float2 ld_cluster_f2(uint32_t addr) {
  float2 v;
  asm volatile("ld.shared::cluster.v2.f32 {%0,%1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(addr) : "memory");
  return v;
}

// one token row of a tile: four columns a lane (gated: two columns a lane). `at`: this row's sums in this CTA's shared memory
__device__ __forceinline__ void finish_row(const LinearArgs& a, int64_t row, int tile, uint32_t at, int splits, int lane) {
  float y[4];
  int col, cols;
  if (a.act.kind == kGated) {
    const int g = lane >> 4, j = (lane & 15) * 2;
    col = tile * 64 + 32 * g + j;
    cols = 2;
    float2 p = make_float2(0.0f, 0.0f), u = p;
    for (int r = 0; r < splits; ++r) {
      const uint32_t from = splits > 1 ? map_to_cta(at, r) : at;
      const float2 pr = ld_cluster_f2(from + (64 * g + j) * 4), ur = ld_cluster_f2(from + (64 * g + 32 + j) * 4);
      p.x += pr.x, p.y += pr.y, u.x += ur.x, u.y += ur.y;
    }
    if (a.bias != nullptr && col < a.n) {
      const float2 bp = __ldcg(reinterpret_cast<const float2*>(a.bias + col)), bu = __ldcg(reinterpret_cast<const float2*>(a.bias + a.n + col));
      p.x += bp.x, p.y += bp.y, u.x += bu.x, u.y += bu.y;
    }
    const F2 v = act_gated(F2{p.x, p.y}, F2{u.x, u.y}, a.act);
    y[0] = v.x, y[1] = v.y, y[2] = y[3] = 0.0f;
  } else {
    col = tile * 128 + lane * 4;
    cols = 4;
    float4 p = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    for (int r = 0; r < splits; ++r) {
      const float4 pr = ld_cluster_f4((splits > 1 ? map_to_cta(at, r) : at) + lane * 16);
      p.x += pr.x, p.y += pr.y, p.z += pr.z, p.w += pr.w;
    }
    if (a.bias != nullptr && col < a.n) {
      const float4 b = __ldcg(reinterpret_cast<const float4*>(a.bias + col));
      p.x += b.x, p.y += b.y, p.z += b.z, p.w += b.w;
    }
    F2 lo = {p.x, p.y}, hi = {p.z, p.w};
    if (a.act.kind == kLinear) lo = act_of<kLinear>(lo, a.act), hi = act_of<kLinear>(hi, a.act);
    else if (a.act.kind == kSigmoid) lo = act_of<kSigmoid>(lo, a.act), hi = act_of<kSigmoid>(hi, a.act);
    else lo = act_of<kGelu>(lo, a.act), hi = act_of<kGelu>(hi, a.act);
    y[0] = lo.x, y[1] = lo.y, y[2] = hi.x, y[3] = hi.y;
  }
  const bool in = col < a.n;  // (n is a multiple of 8: a lane's columns are all inside or all outside)
  if (a.residual != nullptr && in) {
    const __nv_bfloat16* r = a.residual + row * a.residual_stride + col;
    const uint32_t r0 = __ldcg(reinterpret_cast<const uint32_t*>(r));
    y[0] += __uint_as_float(r0 << 16), y[1] += __uint_as_float(r0 & 0xffff0000u);
    if (cols == 4) {
      const uint32_t r1 = __ldcg(reinterpret_cast<const uint32_t*>(r) + 1);
      y[2] += __uint_as_float(r1 << 16), y[3] += __uint_as_float(r1 & 0xffff0000u);
    }
  }
  if (a.out != nullptr) {
    if (!in) return;
    __nv_bfloat16* o = a.out + row * a.out_stride + col;
    if (cols == 4) *reinterpret_cast<uint2*>(o) = make_uint2(pack_bf16x2(y[0], y[1]), pack_bf16x2(y[2], y[3]));
    else *reinterpret_cast<uint32_t*>(o) = pack_bf16x2(y[0], y[1]);
    return;
  }
  // a block of 32 columns is 8 lanes (gated: 16)
  float amax = fmaxf(fmaxf(fabsf(y[0]), fabsf(y[1])), fmaxf(fabsf(y[2]), fabsf(y[3])));
  for (int off = 1; off < 32 / cols; off <<= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, off));
  const int e = linear_scale(amax);
  const float inv = e8m0_value(static_cast<uint32_t>(254 - e));
  if (!in) return;
  uint8_t* o = a.out_codes + row * a.n + col;
  if (cols == 4) *reinterpret_cast<uint32_t*>(o) = pack_e4m3x4(y[0] * inv, y[1] * inv, y[2] * inv, y[3] * inv);
  else *reinterpret_cast<uint16_t*>(o) = static_cast<uint16_t>(cvt_e4m3x2(y[0] * inv, y[1] * inv));
  if ((col & 31) == 0) a.out_scales[row * (a.n / 32) + col / 32] = static_cast<uint8_t>(e);
}

template <int BM>
__global__ void __launch_bounds__(256, LinearCfg<BM>::kCtasPerSm)
    linear_tc_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ LinearArgs args, int splits, int n_blocks,
                     int32_t* status) {
  using C = LinearCfg<BM>;
  extern __shared__ uint8_t smem_raw[];
  __shared__ __align__(8) uint64_t bar_full[C::kStages];   // weight image and token rows of the stage have landed
  __shared__ __align__(8) uint64_t bar_empty[C::kStages];  // the MMAs that read it have completed
  __shared__ __align__(8) uint64_t bar_sfull[C::kSfSlots];    // the scales of the group are in shared memory
  __shared__ __align__(8) uint64_t bar_sf[C::kSfSlots];       // they are in tensor memory
  __shared__ __align__(8) uint64_t bar_set[kSfSets];       // the MMAs that read the set have completed
  __shared__ __align__(8) uint64_t bar_tfull;
  __shared__ __align__(8) uint64_t bar_drain[2];
  __shared__ uint32_t tmem_base_slot;
  __shared__ int abort_flag;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t tiles = (smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t* const tiles_ptr = smem_raw + (tiles - smem_u32(smem_raw));
  volatile int* abort_v = &abort_flag;
  pdl_launch_dependents();
  if (threadIdx.x == 0) {
    abort_flag = 0;
    for (int s = 0; s < C::kStages; ++s) {
      mbar_init(smem_u32(&bar_full[s]), 1);
      mbar_init(smem_u32(&bar_empty[s]), 1);
    }
    for (int j = 0; j < C::kSfSlots; ++j) {
      mbar_init(smem_u32(&bar_sfull[j]), 2);  // the byte count of the weights' atoms, the tokens' atoms
      mbar_init(smem_u32(&bar_sf[j]), 1);
    }
    for (int j = 0; j < kSfSets; ++j) mbar_init(smem_u32(&bar_set[j]), 1);
    mbar_init(smem_u32(&bar_tfull), 1);
    mbar_init(smem_u32(&bar_drain[0]), 1);
    mbar_init(smem_u32(&bar_drain[1]), 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    fence_proxy_async();
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_base_slot)),
                 "r"(static_cast<uint32_t>(C::kTmemCols))
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  const int unit = static_cast<int>(blockIdx.x) / splits, rank = static_cast<int>(blockIdx.x) % splits;
  const int tile = unit / n_blocks, block = unit % n_blocks;
  const int64_t row0 = static_cast<int64_t>(block) * BM;
  const int kt0 = static_cast<int>(static_cast<int64_t>(args.tiles_k) * rank / splits);
  const int kt1 = static_cast<int>(static_cast<int64_t>(args.tiles_k) * (rank + 1) / splits);
  // What the ring will load first, asked into L2 while the launch in front still runs. (The CTA's whole share at once delays these first
  // bytes: 10.4 -> 11.6 us for one row 6144 -> 6144.)
  if (warp == 0 && lane == 0) {
    const int64_t at = static_cast<int64_t>(tile) * args.tiles_k + kt0;
    const int n = kt1 - kt0 < C::kStages ? kt1 - kt0 : C::kStages;
    l2_prefetch_bulk(args.atoms + at * kAtomBytes, static_cast<uint32_t>(n) * kAtomBytes);
    for (int kt = 0; kt < n; ++kt) l2_prefetch_bulk(args.tiles + (at + kt) * kLinearImageBytes, kLinearImageBytes);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = tmem_base_slot;
  pdl_wait();
  LinearArgs a = args;
  launder(a.tiles);
  launder(a.atoms);
  launder(a.scales);
  launder(a.bias);
  launder(a.residual);

  if (warp == 0) {
    scales_first_wait();
    if (lane == 0) {  // ------------------------------------------------ code producer
      const uint8_t* w_src = a.tiles + (static_cast<int64_t>(tile) * a.tiles_k + kt0) * kLinearImageBytes;
      uint32_t it = 0, s = 0, ph = 1u;
      bool ok = true;
      for (int kt = kt0; kt < kt1; ++kt, ++it, w_src += kLinearImageBytes) {
        if (!mbar_wait(smem_u32(&bar_empty[s]), ph, abort_v, status)) { ok = false; break; }
        const uint32_t full = smem_u32(&bar_full[s]), base = tiles + s * C::kStageBytes;
        mbar_arrive_expect_tx(full, C::kStageBytes);
        bulk_load(base, w_src, kLinearImageBytes, full);
        tma_load_2d(base + C::kTokOff, &map_x, kt * 128, static_cast<int>(row0), full);
        if (++s == C::kStages) { s = 0; ph ^= 1u; }
      }
      if (!ok) drain_copies(bar_full, it, C::kStages);
    }
  } else if (warp == 1) {
    // ------------------------------------------------ MMA issue: E4M3 x E4M3, UE8M0 scales, M = 128, N = BM
    constexpr uint32_t kIdesc = (static_cast<uint32_t>(BM >> 3) << 17) | (1u << 23) | (8u << 24);
    uint32_t s = 0, ph = 0, slot = 0, sph = 0, set = 0;
    bool ok = true, ready = false;
    for (int kt = kt0; kt < kt1 && ok; kt += kSfGroup) {
      if (!warp_wait(smem_u32(&bar_sf[slot]), sph, abort_v, status)) { ok = false; break; }
      if (++slot == C::kSfSlots) { slot = 0; sph ^= 1u; }
      const int n = kt1 - kt < kSfGroup ? kt1 - kt : kSfGroup;
      uint32_t t_sfw = tmem_base + BM + set * kSfGroup * C::kSfCols;
#pragma unroll 1
      for (int d = 0; d < n; ++d, t_sfw += C::kSfCols) {
        if (!__all_sync(0xffffffffu, ready || mbar_wait(smem_u32(&bar_full[s]), ph, abort_v, status))) { ok = false; break; }
        tc_fence_after();
        const uint32_t w_lo = (tiles + s * C::kStageBytes) >> 4, x_lo = w_lo + (C::kTokOff >> 4), empty = smem_u32(&bar_empty[s]);
        const uint32_t t_sfx = t_sfw + C::kSfCols / 2;
        if (++s == C::kStages) { s = 0; ph ^= 1u; }
        ready = mbar_test(smem_u32(&bar_full[s]), ph);
        if (elect_one()) {
          tc_mma_mxf8_lo<2>(tmem_base, w_lo, x_lo, kIdesc, t_sfw, t_sfx, static_cast<uint32_t>(kt + d != kt0));
          tc_mma_mxf8_lo<1>(tmem_base, w_lo + 2, x_lo + 2, kIdesc | (1u << 29) | (1u << 4), t_sfw, t_sfx);
          tc_mma_mxf8_lo<1>(tmem_base, w_lo + 4, x_lo + 4, kIdesc | (2u << 29) | (2u << 4), t_sfw, t_sfx);
          tc_mma_mxf8_lo<1>(tmem_base, w_lo + 6, x_lo + 6, kIdesc | (3u << 29) | (3u << 4), t_sfw, t_sfx);
          tc_commit(empty);
          if (d == n - 1) tc_commit(smem_u32(&bar_set[set]));
        }
        __syncwarp();
      }
      if (++set == kSfSets) set = 0;
    }
    if (ok && elect_one()) tc_commit(smem_u32(&bar_tfull));
    if (__any_sync(0xffffffffu, *abort_v != 0) && elect_one()) drain_tcgen05(smem_u32(&bar_drain[0]));
  } else if (warp == 2) {
    // ------------------------------------------------ scale copies into tensor memory
    uint32_t slot = 0, ph = 0, set = 0, set_ph = 1u;
    for (int kt = kt0; kt < kt1; kt += kSfGroup) {
      if (!__all_sync(0xffffffffu, mbar_wait(smem_u32(&bar_sfull[slot]), ph, abort_v, status) &&
                                       mbar_wait(smem_u32(&bar_set[set]), set_ph, abort_v, status)))
        break;
      tc_fence_after();
      const int n = kt1 - kt < kSfGroup ? kt1 - kt : kSfGroup;
      const uint32_t w_atom = (tiles + C::kSfOff + slot * C::kSfSlotBytes) >> 4, x_atom = w_atom + (kSfGroup * kAtomBytes >> 4);
      const uint32_t t_sfw = tmem_base + BM + set * kSfGroup * C::kSfCols, t_sfx = t_sfw + C::kSfCols / 2;
      if (elect_one()) {
        for (int d = 0; d < n; ++d) {
          tc_cp_scales_lo(t_sfw + d * C::kSfCols, w_atom + d * (kAtomBytes >> 4));
#pragma unroll
          for (int h = 0; h < C::kAtoms; ++h) tc_cp_scales_lo(t_sfx + d * C::kSfCols + 4 * h, x_atom + (d * C::kAtoms + h) * (kAtomBytes >> 4));
        }
        tc_commit(smem_u32(&bar_sf[slot]));
      }
      __syncwarp();
      if (++slot == C::kSfSlots) { slot = 0; ph ^= 1u; }
      if (++set == kSfSets) { set = 0; set_ph ^= 1u; }
    }
    if (__any_sync(0xffffffffu, *abort_v != 0) && elect_one()) drain_tcgen05(smem_u32(&bar_drain[1]));
  } else if (warp == 3) {
    // ------------------------------------------------ scale producer: lane l writes an atom's 16 bytes of rows l, l + 32, l + 64, l + 96.
    // A group's bytes are asked for two groups ahead.
    constexpr int kRows = (BM + 31) / 32;
    const RowScales scales(a.scales, a.m, a.k);
    const int64_t row = BM >= 32 || lane < BM ? row0 + lane : a.m;  // (BM = 16: the other lanes' rows are beyond the last)
    uint32_t even[kRows][5] = {}, odd[kRows][5] = {};
    const auto fetch = [&](int kt, uint32_t (&v)[kRows][5]) {
      if (kt < kt1) scales.load(row, kt, v);
    };
    uint32_t slot = 0, ph = 1u, it = 0;
    bool ok = true;
    const auto group = [&](int kt, uint32_t (&v)[kRows][5]) {
      if (kt >= kt1 || !ok) return;
      if (!warp_wait(smem_u32(&bar_sf[slot]), ph, abort_v, status)) { ok = false; return; }
      const uint32_t sfull = smem_u32(&bar_sfull[slot]), at = C::kSfOff + slot * C::kSfSlotBytes;
      if (lane == 0) {
        const uint32_t bytes = (kt1 - kt < kSfGroup ? kt1 - kt : kSfGroup) * kAtomBytes;
        mbar_arrive_expect_tx(sfull, bytes);
        bulk_load(tiles + at, a.atoms + (static_cast<int64_t>(tile) * a.tiles_k + kt) * kAtomBytes, bytes, sfull);
      }
      if (it++ == 0) scales_first_arrive();
      scales.tiles(row, kt, v);
      uint4* cells = reinterpret_cast<uint4*>(tiles_ptr + at + kSfGroup * kAtomBytes) + lane;
#pragma unroll
      for (int d = 0; d < kSfGroup; ++d)
#pragma unroll
        for (int h = 0; h < C::kAtoms; ++h)
          cells[(d * C::kAtoms + h) * 32] = make_uint4(v[4 * h][d], kRows > 1 ? v[(4 * h + 1) % kRows][d] : 0u,
                                                       kRows > 2 ? v[(4 * h + 2) % kRows][d] : 0u, kRows > 2 ? v[(4 * h + 3) % kRows][d] : 0u);
      fence_proxy_async();
      __syncwarp();
      if (lane == 0) mbar_arrive(sfull);
      fetch(kt + 2 * kSfGroup, v);
      if (++slot == C::kSfSlots) { slot = 0; ph ^= 1u; }
    };
    fetch(kt0, even);
    fetch(kt0 + kSfGroup, odd);
    for (int kt = kt0; kt < kt1 && ok; kt += 2 * kSfGroup) {
      group(kt, even);
      group(kt + kSfGroup, odd);
    }
    if (!ok && lane == 0) drain_copies(bar_sfull, it, C::kSfSlots);
  } else {
    // ------------------------------------------------ the part: lane = weight row, column = token. All copies have landed and all MMAs have
    // read them (the last commit), so the ring's memory is free.
    const int q = warp & 3;
    float* mine = reinterpret_cast<float*>(tiles_ptr) + q * 32 + lane;
    if (__all_sync(0xffffffffu, mbar_wait(smem_u32(&bar_tfull), 0, abort_v, status))) {
      tc_fence_after();
      const uint32_t t_acc = tmem_base + (static_cast<uint32_t>(q * 32) << 16);
#pragma unroll 1
      for (int c0 = 0; c0 < BM && row0 + c0 < a.m; c0 += 16) {
        uint32_t v[16];
        tc_ld16(t_acc + c0, v);
#pragma unroll
        for (int j = 0; j < 16; ++j) mine[(c0 + j) * C::kSumRow] = __uint_as_float(v[j]);
      }
    }
  }

  // ---------------------------------------------------------------- the block's rows, shared out over the CTAs of the cluster
  tc_fence_before();
  __syncthreads();
  if (splits > 1) cluster_sync_all();
  const int rows = static_cast<int>(a.m - row0 < BM ? a.m - row0 : BM);
  if (!abort_flag)
    for (int t = rank * 8 + warp; t < rows; t += 8 * splits) finish_row(a, row0 + t, tile, tiles + t * C::kSumRow * 4, splits, lane);
  __syncwarp();
  if (splits > 1) cluster_sync_all();  // nobody leaves while its parts are read
  if (warp == 1) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base),
                 "r"(static_cast<uint32_t>(C::kTmemCols))
                 : "memory");
  }
}

template <int BM>
static int launch_linear_tc(const LinearArgs& a, int splits, int32_t* status, cudaStream_t stream) {
  using C = LinearCfg<BM>;
  static PerDeviceOnce once;
  int r = once.run([] {
    return static_cast<int>(cudaFuncSetAttribute(linear_tc_kernel<BM>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmemBytes));
  });
  if (r) return r;
  CUtensorMap mx;
  if ((r = make_map(&mx, a.codes, static_cast<uint64_t>(a.k), static_cast<uint64_t>(a.m), BM))) return r;
  const int64_t n_blocks = (a.m + BM - 1) / BM, ctas = n_blocks * a.tiles_n * splits;
  if (ctas > 0x7fffffff) return B200MOE_E_ARG;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(ctas));
  cfg.blockDim = dim3(256);
  cfg.dynamicSmemBytes = C::kSmemBytes;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = splits;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = splits > 1 ? 2 : 1;
  return static_cast<int>(cudaLaunchKernelEx(&cfg, linear_tc_kernel<BM>, mx, a, splits, static_cast<int>(n_blocks), status));
}

// bm: 16, 32, 64, 128 or 256 token rows a block; splits: CTAs along K, 1 to 8 and at most the K-tiles
int linear_tc(const LinearArgs& a, int bm, int splits, int32_t* status, cudaStream_t stream) {
  switch (bm) {
    case 16: return launch_linear_tc<16>(a, splits, status, stream);
    case 32: return launch_linear_tc<32>(a, splits, status, stream);
    case 64: return launch_linear_tc<64>(a, splits, status, stream);
    case 128: return launch_linear_tc<128>(a, splits, status, stream);
  }
  return launch_linear_tc<256>(a, splits, status, stream);
}

int set_wait_limit_linear_tc(unsigned long long ns) { return set_wait_limit_here(ns); }

}  // namespace b200moe
