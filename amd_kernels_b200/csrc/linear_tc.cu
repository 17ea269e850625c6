// The MXFP8 product for few rows: tcgen05.mma kind::mxf8f6f4 block-scaled with the weight tile as the 128-row M operand and a block of
// BM token rows as N, so that one pass over the weights serves the whole block.
//
// What bounds it: the weight stream (HBM; one row 6144 -> 4096 takes 8.3 us, 4.0 at the copy rate; a call without work takes 3 to 4). One CTA =
// (weight tile, token block, part of K). K is split over the CTAs of a cluster until there are enough of them to keep every SM loading;
// each adds its part in tensor memory and writes it to its shared memory; after a cluster barrier the CTAs share out the block's
// rows: the parts of a row are fetched and added in the order of K, then bias, activation, residual and the only rounding. No workspace, no atomics, one launch, sums in a fixed order. What bounds the end of a call is distributed
// shared memory: 48 KB into a CTA (128 rows split by 4) take 8000 cycles, fetched by 16 bytes a lane or sent by 4 alike.
//
//   warp 0     code producer: the weight image (one bulk copy of consecutive HBM bytes) and the token rows (TMA)
//   warp 1     tensor memory; issues the MMAs, the whole warp around one elected lane
//   warp 2     scales: shared memory -> tensor memory
//   warp 3     scale producer: the weights' atoms (bulk copy); the tokens' from row-major global memory through registers
//   warps 4-7  the sum out of tensor memory; all warps take part in what follows
//
// QUANT, for a few bf16 rows: there is no launch that quantises them. Warps 4-7, idle until the sum is there, quantise the block's rows
// K-tile by K-tile into the stage, codes and scale atom, while the weights stream; every CTA does it again for its weight tile (the
// rows are a few hundred KB in L2). A stage is then one barrier: image, weight atom and tokens. It saves a launch, which counts where the host
// is the bound (two eager calls 15 us, the one 9.2 to 16 to 4096 columns, 17.7 to 50 to 12288); on the device the repeated work mostly costs
// more than a launch in front. K = 6144, captured, us inside / quantised in front / from MXFP8 rows: 16 rows to 4096 columns 8.8 / 9.3 / 7.7,
// to 12288 17.6 / 14.1 / 12.7; 64 rows 16.1 / 11.6 / 9.8 and 49.6 / 16.6 / 16.8; one row 10.5 / 8.4 / 7.2 and 24.6 / 13.5 / 12.9 (a zero takes
// the slow way through the scale's division, so rows of zeros and the empty ones of a block cost most: 16 rows to 12288 17.3, 27.7 with 15
// of them zero).
//
// Weights of more tiles than CTAs run at once (37888 rows) go without a split, in rounds: one row 6144 -> 131072 120 us (127 at the copy rate), 64
// rows 133, 128 rows 159; just above the limit a round of few tiles is the price: one row -> 37888 39.6, -> 38016 48.4.
#include "linear.cuh"
#include "tc_pair.cuh"

namespace b200moe {

template <int BM, bool QUANT = false>
struct LinearCfg {
  static constexpr int kTokOff = kLinearImageBytes;               // token rows behind the weight image
  static constexpr int kStageBytes = kTokOff + BM * 128;
  static constexpr int kCtasPerSm = 2;                            // one's start and end under the other's stream
  static constexpr int kStages = BM > 64 ? 3 : BM > 32 ? 4 : 5;
  static constexpr int kSfSlots = BM == 32 ? 2 : 3;               // groups of scales in shared memory; QUANT: a slot a stage
  static constexpr int kSfOff = kStages * kStageBytes;
  static constexpr int kSfSlotBytes = kSfGroup * 2 * kAtomBytes;  // weight atoms of the group, then token atoms
  static constexpr int kSumRow = 132;                             // floats of a token's 128 columns in the parts (alias the ring)
  static constexpr int kSmemBytes = kSfOff + (QUANT ? kStages * 2 * kAtomBytes : kSfSlots * kSfSlotBytes) + 1024;
  static constexpr int kSfCols = 8;                               // tensor memory columns of a K-tile's scales: 4 weights, 4 tokens
  static constexpr int kColsUsed = BM + kSfSets * kSfGroup * kSfCols;
  static constexpr int kTmemCols = kColsUsed <= 128 ? 128 : 256;
  static_assert(BM * kSumRow * 4 <= kSfOff, "the parts fit the ring");
  static_assert(kSmemBytes <= 227 * 1024 / kCtasPerSm - 1024 && kTmemCols * kCtasPerSm <= 512, "shared and tensor memory");
  // A CTA of the next launch may be there early. It must not hold tensor memory that one of this launch has yet to get: no third one of these
  // fits an SM (nor any of the layer's kernels, which take more shared memory) until one of the two has left.
  static_assert(3 * kSmemBytes > 227 * 1024, "three CTAs on an SM");
};

// (neither volatile nor ordered by a memory clobber: the loads of a row's parts have to be in flight together; what orders them is the
// barrier in front, behind which their address is laundered)
template <bool CLUSTER>
__device__ __forceinline__ float4 ld_part(uint32_t addr) {
  float4 v;
  if (CLUSTER) asm("ld.shared::cluster.v4.f32 {%0,%1,%2,%3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr));
  else asm("ld.shared.v4.f32 {%0,%1,%2,%3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr));
  return v;
}

// The rows of the block that fall to this warp (every `step`-th from `first` on): the parts of a row are added in the order of K, then bias,
// activation, residual and the only rounding. A lane has four of the tile's 128 columns; gated, lanes 0-7 and 16-23 have the gates of
// four output columns and take the ups from the lanes 8 above. `parts`: the sums in this CTA's shared memory, SUM_ROW floats a row. (The
// splits are a template's: with a branch around each load the loads of a row wait for one another, 450 cycles each.)
template <int SUM_ROW, int SPLITS>
__device__ __forceinline__ void finish_rows(const LinearArgs& a, int64_t row0, int rows, int first, int tile, uint32_t parts, int lane) {
  const bool gated = a.act.kind == kGated;
  const int col = gated ? tile * 64 + 32 * (lane >> 4) + (lane & 7) * 4 : tile * 128 + lane * 4;
  const bool up = gated && (lane & 8);
  const bool in = col < a.n && !up;  // (n is a multiple of 8: a lane's columns are all inside or all outside)
  float4 bias = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  if (a.bias != nullptr && col < a.n) bias = __ldcg(reinterpret_cast<const float4*>(a.bias + (up ? a.n : 0) + col));
  uint32_t from[SPLITS];
#pragma unroll
  for (int r = 0; r < SPLITS; ++r) from[r] = (SPLITS > 1 ? map_to_cta(parts, r) : parts) + lane * 16;
#pragma unroll 2
  for (int t = first; t < rows; t += 8 * SPLITS) {
    const int64_t row = row0 + t;
    float4 part[SPLITS];
#pragma unroll
    for (int r = 0; r < SPLITS; ++r) part[r] = ld_part<(SPLITS > 1)>(from[r] + t * SUM_ROW * 4);
    uint2 res = make_uint2(0u, 0u);
    if (a.residual != nullptr && in) res = __ldcg(reinterpret_cast<const uint2*>(a.residual + row * a.residual_stride + col));
    float4 p = part[0];
#pragma unroll
    for (int r = 1; r < SPLITS; ++r) p.x += part[r].x, p.y += part[r].y, p.z += part[r].z, p.w += part[r].w;
    F2 y[2] = {F2{p.x, p.y} + F2{bias.x, bias.y}, F2{p.z, p.w} + F2{bias.z, bias.w}};
    if (gated) {
      const F2 u[2] = {{__shfl_down_sync(0xffffffffu, y[0].x, 8), __shfl_down_sync(0xffffffffu, y[0].y, 8)},
                       {__shfl_down_sync(0xffffffffu, y[1].x, 8), __shfl_down_sync(0xffffffffu, y[1].y, 8)}};
      act_gated(y, u, a.act);
    } else if (a.act.kind == kLinear) {
      act_of<kLinear>(y, a.act);
    } else if (a.act.kind == kSigmoid) {
      act_of<kSigmoid>(y, a.act);
    } else {
      act_of<kGelu>(y, a.act);
    }
    F2 lo = y[0], hi = y[1];
    if (a.residual != nullptr) {
      lo = lo + F2{__uint_as_float(res.x << 16), __uint_as_float(res.x & 0xffff0000u)};
      hi = hi + F2{__uint_as_float(res.y << 16), __uint_as_float(res.y & 0xffff0000u)};
    }
    if (a.out != nullptr) {
      if (in) *reinterpret_cast<uint2*>(a.out + row * a.out_stride + col) = make_uint2(pack_bf16x2(lo.x, lo.y), pack_bf16x2(hi.x, hi.y));
    } else {  // a block of 32 columns is 8 neighbouring lanes
      float amax = fmaxf(fmaxf(fabsf(lo.x), fabsf(lo.y)), fmaxf(fabsf(hi.x), fabsf(hi.y)));
#pragma unroll
      for (int off = 1; off < 8; off <<= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, off));
      const int e = linear_scale(amax);
      const float inv = e8m0_value(static_cast<uint32_t>(254 - e));
      if (in) {
        *reinterpret_cast<uint32_t*>(a.out_codes + row * a.n + col) = pack_e4m3x4(lo.x * inv, lo.y * inv, hi.x * inv, hi.y * inv);
        if ((lane & 7) == 0) a.out_scales[row * (a.n / 32) + col / 32] = static_cast<uint8_t>(e);
      }
    }
  }
}

template <int BM, bool QUANT>
__global__ void __launch_bounds__(256, LinearCfg<BM>::kCtasPerSm)
    linear_tc_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ LinearArgs args, int splits, int n_blocks,
                     int32_t* status) {
  using C = LinearCfg<BM, QUANT>;
  extern __shared__ uint8_t smem_raw[];
  __shared__ __align__(8) uint64_t bar_full[C::kStages];   // weight image and token rows of the stage have landed
  __shared__ __align__(8) uint64_t bar_empty[C::kStages];  // the MMAs that read it have completed
  __shared__ __align__(8) uint64_t bar_sfull[C::kSfSlots];    // the scales of the group are in shared memory
  __shared__ __align__(8) uint64_t bar_sf[QUANT ? C::kStages : C::kSfSlots];  // they (QUANT: the stage's) are in tensor memory
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
      mbar_init(smem_u32(&bar_full[s]), QUANT ? 5 : 1);  // the byte count; QUANT: four warps' tokens too
      mbar_init(smem_u32(&bar_empty[s]), 1);
      if (QUANT) mbar_init(smem_u32(&bar_sf[s]), 1);
    }
    for (int j = 0; j < C::kSfSlots; ++j) {
      mbar_init(smem_u32(&bar_sfull[j]), 2);  // the byte count of the weights' atoms, the tokens' atoms
      if (!QUANT) mbar_init(smem_u32(&bar_sf[j]), 1);
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
    for (int kt = 0; kt < n; ++kt) {
      l2_prefetch_bulk(args.tiles + (at + kt) * kLinearImageBytes, kLinearImageBytes);
      if (!QUANT) tma_prefetch_2d(&map_x, (kt0 + kt) * 128, static_cast<int>(row0));
    }
  }
  if (!QUANT && threadIdx.x == 32) prefetch_map(&map_x);
  if (!QUANT && warp == 3) RowScales(args.scales, args.m, args.k).prefetch<(BM + 31) / 32>(row0 + lane, kt0);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = tmem_base_slot;
  pdl_wait();
  LinearArgs a = args;
  launder(a.tiles);
  launder(a.atoms);
  launder(a.scales);
  launder(a.x);
  launder(a.bias);
  launder(a.residual);

  if (QUANT && warp == 0) {
    if (lane == 0) {  // ------------------------------------------------ QUANT: weights, images and atoms
      const int64_t at = static_cast<int64_t>(tile) * a.tiles_k;
      uint32_t it = 0, s = 0, ph = 1u;
      bool ok = true;
      for (int kt = kt0; kt < kt1; ++kt, ++it) {
        if (!mbar_wait(smem_u32(&bar_empty[s]), ph, abort_v, status)) { ok = false; break; }
        const uint32_t full = smem_u32(&bar_full[s]);
        mbar_arrive_expect_tx(full, kLinearTileBytes);
        bulk_load(tiles + s * C::kStageBytes, a.tiles + (at + kt) * kLinearImageBytes, kLinearImageBytes, full);
        bulk_load(tiles + C::kSfOff + s * 2 * kAtomBytes, a.atoms + (at + kt) * kAtomBytes, kAtomBytes, full);
        if (++s == C::kStages) { s = 0; ph ^= 1u; }
      }
      if (!ok) drain_copies(bar_full, it, C::kStages);
    }
  } else if (QUANT && warp == 1) {
    // ------------------------------------------------ QUANT: MMA issue
    constexpr uint32_t kIdesc = (static_cast<uint32_t>(BM >> 3) << 17) | (1u << 23) | (8u << 24);
    uint32_t s = 0, ph = 0;
    bool ok = true;
    for (int kt = kt0; kt < kt1; ++kt) {
      if (!warp_wait(smem_u32(&bar_sf[s]), ph, abort_v, status)) { ok = false; break; }
      tc_fence_after();
      const uint32_t w_lo = (tiles + s * C::kStageBytes) >> 4, x_lo = w_lo + (C::kTokOff >> 4);
      const uint32_t t_sfw = tmem_base + BM + s * C::kSfCols, t_sfx = t_sfw + C::kSfCols / 2;
      if (elect_one()) {
        tc_mma_mxf8_lo<2>(tmem_base, w_lo, x_lo, kIdesc, t_sfw, t_sfx, static_cast<uint32_t>(kt != kt0));
        tc_mma_mxf8_lo<1>(tmem_base, w_lo + 2, x_lo + 2, kIdesc | (1u << 29) | (1u << 4), t_sfw, t_sfx);
        tc_mma_mxf8_lo<1>(tmem_base, w_lo + 4, x_lo + 4, kIdesc | (2u << 29) | (2u << 4), t_sfw, t_sfx);
        tc_mma_mxf8_lo<1>(tmem_base, w_lo + 6, x_lo + 6, kIdesc | (3u << 29) | (3u << 4), t_sfw, t_sfx);
        tc_commit(smem_u32(&bar_empty[s]));
      }
      __syncwarp();
      if (++s == C::kStages) { s = 0; ph ^= 1u; }
    }
    if (ok && elect_one()) tc_commit(smem_u32(&bar_tfull));
    if (__any_sync(0xffffffffu, *abort_v != 0) && elect_one()) drain_tcgen05(smem_u32(&bar_drain[0]));
  } else if (QUANT && warp == 2) {
    // ------------------------------------------------ QUANT: scale copies (the set of a stage is free once the stage is)
    uint32_t s = 0, ph = 0;
    for (int kt = kt0; kt < kt1; ++kt) {
      if (!warp_wait(smem_u32(&bar_full[s]), ph, abort_v, status)) break;
      tc_fence_after();
      const uint32_t atoms = (tiles + C::kSfOff + s * 2 * kAtomBytes) >> 4, t_sfw = tmem_base + BM + s * C::kSfCols;
      if (elect_one()) {
        tc_cp_scales_lo(t_sfw, atoms);
        tc_cp_scales_lo(t_sfw + C::kSfCols / 2, atoms + (kAtomBytes >> 4));
        tc_commit(smem_u32(&bar_sf[s]));
      }
      __syncwarp();
      if (++s == C::kStages) { s = 0; ph ^= 1u; }
    }
    if (__any_sync(0xffffffffu, *abort_v != 0) && elect_one()) drain_tcgen05(smem_u32(&bar_drain[1]));
  } else if (QUANT && warp == 3) {
  } else if (!QUANT && warp == 0) {
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
  } else if (!QUANT && warp == 1) {
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
  } else if (!QUANT && warp == 2) {
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
          tc_cp_scales_lo(t_sfx + d * C::kSfCols, x_atom + d * (kAtomBytes >> 4));
        }
        tc_commit(smem_u32(&bar_sf[slot]));
      }
      __syncwarp();
      if (++slot == C::kSfSlots) { slot = 0; ph ^= 1u; }
      if (++set == kSfSets) { set = 0; set_ph ^= 1u; }
    }
    if (__any_sync(0xffffffffu, *abort_v != 0) && elect_one()) drain_tcgen05(smem_u32(&bar_drain[1]));
  } else if (!QUANT && warp == 3) {
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
      ++it;
      scales.tiles(row, kt, v);
      uint4* cells = reinterpret_cast<uint4*>(tiles_ptr + at + kSfGroup * kAtomBytes) + lane;
#pragma unroll
      for (int d = 0; d < kSfGroup; ++d)
        cells[d * 32] = make_uint4(v[0][d], kRows > 1 ? v[1 % kRows][d] : 0u, kRows > 2 ? v[2 % kRows][d] : 0u, kRows > 2 ? v[3 % kRows][d] : 0u);
      fence_proxy_async();
      __syncwarp();
      if (lane == 0) mbar_arrive(sfull);
      fetch(kt + 2 * kSfGroup, v);
      if (++slot == C::kSfSlots) { slot = 0; ph ^= 1u; }
    };
    fetch(kt0, even);
    scales_first_arrive();
    fetch(kt0 + kSfGroup, odd);
    for (int kt = kt0; kt < kt1 && ok; kt += 2 * kSfGroup) {
      group(kt, even);
      group(kt + kSfGroup, odd);
    }
    if (!ok && lane == 0) drain_copies(bar_sfull, it, C::kSfSlots);
  } else {
    if (QUANT) {
      // ---------------------------------------------- the block's rows: 16 lanes to a row's 256 bytes of a K-tile, four lanes to a scale
      constexpr int kItems = BM * 16 / 128;
      const int et = threadIdx.x - 128, c = et & 15;
      uint4 next[kItems];
      const auto fetch = [&](int kt) {
#pragma unroll
        for (int i = 0; i < kItems; ++i) {
          const int64_t row = row0 + (i * 128 + et) / 16;
          const int col = kt * 128 + c * 8;
          next[i] = kt < kt1 && row < a.m && col < a.k ? __ldcg(reinterpret_cast<const uint4*>(a.x + row * a.x_stride + col)) : uint4{};
        }
      };
      uint32_t s = 0, ph = 1u;
      fetch(kt0);
      for (int kt = kt0; kt < kt1; ++kt) {
        uint4 now[kItems];
#pragma unroll
        for (int i = 0; i < kItems; ++i) now[i] = next[i];
        fetch(kt + 1);
        if (!warp_wait(smem_u32(&bar_empty[s]), ph, abort_v, status)) break;
        uint8_t* const codes = tiles_ptr + s * C::kStageBytes + C::kTokOff;
        uint8_t* const atom = tiles_ptr + C::kSfOff + s * 2 * kAtomBytes + kAtomBytes;
#pragma unroll
        for (int i = 0; i < kItems; ++i) {
          const int r = (i * 128 + et) / 16;
          float v[8];
          unpack_bf16x8(now[i], v);
          float amax = max3_abs(max3_abs(v[0], v[1], v[2]), max3_abs(v[3], v[4], v[5]), max3_abs(v[6], v[7], 0.0f));
          amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
          amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
          const int e = linear_scale(amax);
          const float inv = e8m0_value(static_cast<uint32_t>(254 - e));
          *reinterpret_cast<uint2*>(codes + r * 128 + (((c >> 1) ^ (r & 7)) << 4) + (c & 1) * 8) =
              make_uint2(pack_e4m3x4(v[0] * inv, v[1] * inv, v[2] * inv, v[3] * inv), pack_e4m3x4(v[4] * inv, v[5] * inv, v[6] * inv, v[7] * inv));
          uint32_t sc = static_cast<uint32_t>(e);
          sc |= __shfl_down_sync(0xffffffffu, sc, 4) << 8;
          sc |= __shfl_down_sync(0xffffffffu, sc, 8) << 16;
          if (c == 0) *reinterpret_cast<uint32_t*>(atom + atom_offset(r, 0)) = sc;
        }
        fence_proxy_async();
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&bar_full[s]));
        if (++s == C::kStages) { s = 0; ph ^= 1u; }
      }
    }
    // ------------------------------------------------ the part: lane = weight row, column = token. All copies have landed and all MMAs have
    // read them (the last commit), so the ring's memory is free.
    const int q = warp & 3;
    float* mine = reinterpret_cast<float*>(tiles_ptr) + q * 32 + lane;
    if (__all_sync(0xffffffffu, mbar_wait(smem_u32(&bar_tfull), 0, abort_v, status))) {
      tc_fence_after();
      const uint32_t t_acc = tmem_base + (static_cast<uint32_t>(q * 32) << 16);
      constexpr int kAtOnce = BM < 32 ? BM : 32;
#pragma unroll 1
      for (int c0 = 0; c0 < BM && row0 + c0 < a.m; c0 += kAtOnce) {
        uint32_t v[kAtOnce];
        if constexpr (BM < 32) tc_ld16(t_acc + c0, v);
        else tc_ld32(t_acc + c0, v);
#pragma unroll
        for (int j = 0; j < kAtOnce; ++j) mine[(c0 + j) * C::kSumRow] = __uint_as_float(v[j]);
      }
    }
  }

  // ---------------------------------------------------------------- the block's rows, shared out over the CTAs of the cluster
  tc_fence_before();
  __syncthreads();
  if (splits > 1) cluster_sync_all();
  const int rows = static_cast<int>(a.m - row0 < BM ? a.m - row0 : BM);
  uint32_t parts = tiles;
  asm volatile("" : "+r"(parts)::"memory");
  if (!abort_flag) {
    const int first = rank * 8 + warp;
    if (splits == 4) finish_rows<C::kSumRow, 4>(a, row0, rows, first, tile, parts, lane);
    else if (splits == 2) finish_rows<C::kSumRow, 2>(a, row0, rows, first, tile, parts, lane);
    else if (splits == 1) finish_rows<C::kSumRow, 1>(a, row0, rows, first, tile, parts, lane);
    else if (splits == 6) finish_rows<C::kSumRow, 6>(a, row0, rows, first, tile, parts, lane);
    else finish_rows<C::kSumRow, 8>(a, row0, rows, first, tile, parts, lane);
  }
  __syncwarp();
  // Nobody leaves while its parts are read. (Relaxed: what has been loaded is in registers, and a release would wait for the stores.)
  if (splits > 1) asm volatile("barrier.cluster.arrive.relaxed.aligned;\nbarrier.cluster.wait.aligned;" ::: "memory");
  if (warp == 1) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base),
                 "r"(static_cast<uint32_t>(C::kTmemCols))
                 : "memory");
  }
}

template <int BM, bool QUANT>
static int configure_linear_tc() {
  static PerDeviceOnce once;
  return once.run([] {
    return static_cast<int>(
        cudaFuncSetAttribute(linear_tc_kernel<BM, QUANT>, cudaFuncAttributeMaxDynamicSharedMemorySize, LinearCfg<BM, QUANT>::kSmemBytes));
  });
}

template <int BM, bool QUANT>
static cudaLaunchConfig_t linear_tc_config(int64_t clusters, int splits, cudaLaunchAttribute (&attr)[2], cudaStream_t stream) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(clusters * splits));
  cfg.blockDim = dim3(256);
  cfg.dynamicSmemBytes = LinearCfg<BM, QUANT>::kSmemBytes;
  cfg.stream = stream;
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = splits;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = splits > 1 ? 2 : 1;
  return cfg;
}

template <int BM, bool QUANT>
static int launch_linear_tc(const LinearArgs& a, int splits, int32_t* status, cudaStream_t stream) {
  int r = configure_linear_tc<BM, QUANT>();
  if (r) return r;
  CUtensorMap mx = {};
  if (!QUANT && (r = make_map(&mx, a.codes, static_cast<uint64_t>(a.k), static_cast<uint64_t>(a.m), BM))) return r;
  const int64_t n_blocks = (a.m + BM - 1) / BM, units = n_blocks * a.tiles_n;
  if (units * splits > 0x7fffffff) return B200MOE_E_ARG;
  cudaLaunchAttribute attr[2];
  const cudaLaunchConfig_t cfg = linear_tc_config<BM, QUANT>(units, splits, attr, stream);
  return static_cast<int>(cudaLaunchKernelEx(&cfg, linear_tc_kernel<BM, QUANT>, mx, a, splits, static_cast<int>(n_blocks), status));
}

// Clusters of [splits] CTAs that run at once on the current device; asked once per device. The occupancy calculation counts one CTA
// an SM for kernels that use tensor memory, whatever their shared memory (it says one at 60 KB too); two run (288 CTAs in clusters of two
// take the time of 192), so its number is doubled.
template <int BM>
static LinearResident resident_clusters() {
  static PerDeviceAnswer<LinearResident> answer;
  return answer.get([](LinearResident& clusters) {
    if (configure_linear_tc<BM, false>()) return false;
    bool all = true;
    for (const int splits : {1, 2, 4, 6, 8}) {
      int got = sm_count();
      cudaLaunchAttribute attr[2];
      const cudaLaunchConfig_t cfg = linear_tc_config<BM, false>(sm_count(), splits, attr, nullptr);
      const bool ok = splits == 1 || cudaOccupancyMaxActiveClusters(&got, linear_tc_kernel<BM, false>, &cfg) == cudaSuccess;
      (void)cudaGetLastError();
      clusters.of[splits] = ok ? LinearCfg<BM>::kCtasPerSm * got : 0;
      all = all && ok;
    }
    return all;
  });
}

LinearResident linear_tc_resident(int bm) {
  return bm == 16 ? resident_clusters<16>() : bm == 32 ? resident_clusters<32>() : bm == 64 ? resident_clusters<64>() : resident_clusters<128>();
}

// bm: 16, 32, 64 or 128 token rows a block (a.x given: 16, 32 or 64); splits: 1, 2, 4, 6 or 8 CTAs along K, at most the K-tiles
int linear_tc(const LinearArgs& a, int bm, int splits, int32_t* status, cudaStream_t stream) {
  switch (bm) {
    case 16: return a.x ? launch_linear_tc<16, true>(a, splits, status, stream) : launch_linear_tc<16, false>(a, splits, status, stream);
    case 32: return a.x ? launch_linear_tc<32, true>(a, splits, status, stream) : launch_linear_tc<32, false>(a, splits, status, stream);
    case 64: return a.x ? launch_linear_tc<64, true>(a, splits, status, stream) : launch_linear_tc<64, false>(a, splits, status, stream);
  }
  return launch_linear_tc<128, false>(a, splits, status, stream);
}

int set_wait_limit_linear_tc(unsigned long long ns) { return set_wait_limit_here(ns); }

}  // namespace b200moe
