// The MXFP8 product for many rows, on CTA pairs: tcgen05.mma.cta_group::2 kind::mxf8f6f4 with M = 256 token rows (two blocks of 128) x
// N = 256 weight rows (two tiles) x K = 32 per instruction, each CTA staging its own 128 token rows and half of the
// weight rows. No multicast.
//
// Unit = (pair of token blocks) x (pair of weight tiles). Two rings: 5 stages of codes, and 2 slots of the scales of four K-tiles that travel
// ahead of them, so that the MMA warp waits for codes and, once in four K-tiles, for scales. The token scales come row-major, as every
// producer of this package writes them: the scale warp turns them into atoms on the way, so no launch in front of the product re-lays them.
//
//   warp 0      code producer (both CTAs): TMA of the CTA's 128 token rows and of its weight rows, counted on the leader's barrier
//   warp 1      tensor memory (both CTAs); in the leader it issues the MMAs for both, the whole warp around one elected lane
//   warp 2      leader: copies the scales into tensor memory in both CTAs, in the same way; partner: tells the leader of its token scales
//   warp 3      scales (both CTAs): the CTA's token rows through registers, the atoms of the weight tiles by TMA
//   warps 4-11  epilogue (both CTAs): thread = one token row, 128 columns. The sums are pulled into registers and the accumulator
//               is handed back; then bias, activation, residual and one rounding, 32 columns at a time. bf16 rows go through a strip of
//               shared memory per warp, pieces of 32 rows x 32 columns: the residual arrives by TMA, two pieces ahead, the result
//               leaves by TMA. (A thread's own 16- or 32-byte pieces of its row cost the shared memory a cycle each, cycles in which the
//               operands of the MMAs wait: with them a residual made 16384 x 6144 -> 6144 28 % slower.)
// 12 warps start with 168 registers; the issuing warpgroup drops to 88, the epilogue's rise to 208 (4 x 88 + 8 x 208 = 12 x 168: the
// exchange must balance inside what the CTA was given at launch). What does not fit the 168 at the start spills: up to 44 bytes stored and 200
// loaded a thread, in all forms.
//
// What bounds it: the tensor pipe for long sums and many rows (4095 x 6144 -> 8192: busy 75 % of the cycles; the rest are the start, the ends
// of units and waits for L2, 1.8 GB of operands at 12.5 TB/s) and the power limit: back to back the clock falls from 1.9 to 1.3 GHz, where
// 16384 x 6144 -> 6144 takes 538 us (2.3 PFLOP/s; 445 us in a short burst, 2.8). A call of few K-tiles is bound by its epilogue and by
// what starting and ending it costs, 11 us in all.
#include "linear.cuh"
#include "tc_pair.cuh"

namespace b200moe {

struct LinearPairCfg {
  static constexpr int kStages = 5;                // code ring (6 stages and no strips were 0 to 1 % faster, 4 were 5 % slower)
  static constexpr int kAhead = 8;                 // K-tiles between a weight tile's way into L2 and into the ring
  static constexpr int kSfSlots = 2;               // groups of scales in shared memory
  static constexpr int kWOff = 128 * 128;          // the CTA's weight tile, behind its 128 token rows
  static constexpr int kStageBytes = 2 * 128 * 128;
  static constexpr int kPieceBytes = 32 * 64;      // an epilogue warp's 32 rows x 32 bf16 columns, 64-byte swizzle
  static constexpr int kStripBytes = 3 * kPieceBytes;  // a warp's: two pieces of residual, one of results
  static constexpr int kStripOff = kStages * kStageBytes;
  static constexpr int kSfOff = kStripOff + 8 * kStripBytes;
  static constexpr int kSfSlotBytes = kSfGroup * 3 * kAtomBytes;  // four token atoms, four atoms of each weight tile
  static constexpr int kBiasOff = kSfOff + kSfSlots * kSfSlotBytes;
  static constexpr int kSmemBytes = kBiasOff + 8 * 128 * 4 + 1024;
  static constexpr int kThreads = 32 * 12;
  static constexpr int kSfCol = 256;               // tensor memory: the accumulator, then 2 sets of 4 x 16 columns
  static constexpr int kTmemCols = 512;
  static_assert(kSmemBytes <= 227 * 1024 && kSfCol + kSfSets * kSfGroup * 16 <= kTmemCols, "shared and tensor memory");
};

__device__ __forceinline__ void tc_mma_mxf8_two(uint32_t d, uint32_t a_lo, uint32_t b_lo, uint32_t idesc, uint32_t sfa, uint32_t sfb,
                                                uint32_t accumulate) {
  asm volatile(
      "{\n.reg .b64 da, db;\n.reg .pred p;\nmov.b64 da, {%1, %7};\nmov.b64 db, {%2, %7};\nsetp.ne.b32 p, %6, 0;\n"
      "tcgen05.mma.cta_group::2.kind::mxf8f6f4.block_scale.scale_vec::1X [%0], da, db, %3, [%4], [%5], p;\n}\n" ::"r"(d),
      "r"(a_lo), "r"(b_lo), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate), "n"(kOperandDescHi)
      : "memory");
}

// Arrival on a barrier of another CTA of the cluster that orders what this thread has seen before it, and the wait that sees it. The
// arrival waits for everything that its thread has in flight, so a thread without loads does it for the scale warp, whose own arrival is
// local: with the scale warp arriving itself a group of four K-tiles took 3400 cycles instead of 2300.
__device__ __forceinline__ void mbar_arrive_release_cluster(uint32_t cluster_addr) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr) : "memory");
}
__device__ __forceinline__ bool mbar_wait_acquire_cluster(uint32_t bar, uint32_t parity, volatile int* abort_flag, int32_t* status) {
  if (!mbar_wait(bar, parity, abort_flag, status)) return false;
  uint32_t ok;  // the phase is complete: this look succeeds at once, and acquires at the writers' scope
  asm volatile(
      "{\n.reg .pred p;\nmbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\nselp.u32 %0, 1, 0, p;\n}\n"
      : "=r"(ok)
      : "r"(bar), "r"(parity)
      : "memory");
  return ok != 0;
}

// The units in groups of 16 pairs of token blocks: a group sweeps the weights once, tile by tile, so that its tokens (4096 rows) and the
// few tiles in work stay in L2 whatever the size of the weights. What the SMs read of L2 (64 bytes a cycle each) comes near what it gives
// them, more where neighbours read the same. Measured back to back, us, groups of 8 / 12 / 16 / 24 / 32: 4095 x 6144 -> 8192
// 178 / 177 / 173 / 172 / 172, 8192 x 6144 -> 4096 gated 343 / 343 / 335 / 336 / 341, 16384 x 6144 -> 6144 548 / 539 / 538 / 547 / 575.
struct LinearUnits {
  static constexpr int kGroup = 16;
  int pairs, steps_n;  // pairs of token blocks, units along N
  __device__ __forceinline__ int total() const { return pairs * steps_n; }
  __device__ __forceinline__ void at(int u, int& pair, int& step) const {
    const int group = u / (kGroup * steps_n), first = group * kGroup, rest = u - group * kGroup * steps_n;
    const int rows = pairs - first < kGroup ? pairs - first : kGroup;
    step = rest / rows;
    pair = first + rest % rows;
  }
};

__device__ __forceinline__ void tma_store_2d(const CUtensorMap* map, int x, int y, uint32_t src) {
  asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%2, %3}], [%1];\ncp.async.bulk.commit_group;" ::"l"(
                   reinterpret_cast<uint64_t>(map)),
               "r"(src), "r"(x), "r"(y)
               : "memory");
}
// until the thread's stores have read their shared memory
__device__ __forceinline__ void tma_store_wait_read() { asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory"); }

template <int KIND, bool MX>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(LinearPairCfg::kThreads, 1)
    linear_pair_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_wc,
                       const __grid_constant__ CUtensorMap map_ws, const __grid_constant__ CUtensorMap map_res,
                       const __grid_constant__ CUtensorMap map_out, const __grid_constant__ LinearArgs args, int32_t* status) {
  using C = LinearPairCfg;
  extern __shared__ uint8_t smem_raw[];
  __shared__ __align__(8) uint64_t bar_full[C::kStages];     // leader: both CTAs' codes of the stage have landed
  __shared__ __align__(8) uint64_t bar_empty[C::kStages];    // in each CTA: the MMAs that read the stage have completed
  __shared__ __align__(8) uint64_t bar_sfull[C::kSfSlots];      // leader: both CTAs' scales of the group are there
  __shared__ __align__(8) uint64_t bar_sf[C::kSfSlots];         // in each CTA: they have been copied to tensor memory
  __shared__ __align__(8) uint64_t bar_relay[C::kSfSlots];   // partner: its token scales of the group are in its shared memory
  __shared__ __align__(8) uint64_t bar_set[kSfSets];         // leader: the MMAs that read the set have completed
  __shared__ __align__(8) uint64_t bar_tfull;                // in each CTA: the unit's accumulator is complete
  __shared__ __align__(8) uint64_t bar_tempty;               // leader: both CTAs' epilogues have read it
  __shared__ __align__(8) uint64_t bar_res[8][2];            // the residual of a piece has landed in half 0 or 1 of the warp's strip
  __shared__ __align__(8) uint64_t bar_drain[2];
  __shared__ uint32_t tmem_base_slot;
  __shared__ int abort_flag;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_rank();
  const bool leader = rank == 0;
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
    for (int j = 0; j < kSfSets; ++j) mbar_init(smem_u32(&bar_set[j]), 1);
    for (int j = 0; j < C::kSfSlots; ++j) {
      mbar_init(smem_u32(&bar_sfull[j]), 3);  // the leader's byte count, the token scales of both CTAs
      mbar_init(smem_u32(&bar_sf[j]), 1);
      mbar_init(smem_u32(&bar_relay[j]), 1);
    }
    mbar_init(smem_u32(&bar_tfull), 1);
    mbar_init(smem_u32(&bar_tempty), 16);  // one arrival per epilogue warp of both CTAs
    for (int i = 0; i < 16; ++i) mbar_init(smem_u32(&bar_res[i >> 1][i & 1]), 1);
    mbar_init(smem_u32(&bar_drain[0]), 1);
    mbar_init(smem_u32(&bar_drain[1]), 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    fence_proxy_async();
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_base_slot)),
                 "r"(static_cast<uint32_t>(C::kTmemCols))
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
  const int n_clusters = static_cast<int>(gridDim.x >> 1), cluster = static_cast<int>(blockIdx.x >> 1);
  const LinearUnits units = {static_cast<int>((args.m + 255) / 256), (args.tiles_n + 1) / 2};
  const int total = units.total(), tiles_k = args.tiles_k;
  int pair, step;
  // what this CTA will load first, into L2 while the launch in front still runs
  if (threadIdx.x == 32) {
    prefetch_map(&map_x);
    prefetch_map(&map_wc);
    prefetch_map(&map_ws);
    if (args.residual != nullptr) prefetch_map(&map_res);
    if (!MX) prefetch_map(&map_out);
  }
  if (cluster < total && (warp == 0 || warp == 3)) {
    units.at(cluster, pair, step);
    const int row = pair * 256 + static_cast<int>(rank) * 128, tile = 2 * step + static_cast<int>(rank), n = tiles_k < C::kAhead ? tiles_k : C::kAhead;
    if (warp == 3) {
      RowScales(args.scales, args.m, args.k).prefetch<4>(row + lane, 0);
    } else if (lane == 0) {
      const int64_t at = static_cast<int64_t>(tile) * tiles_k;
      if (tile < args.tiles_n) l2_prefetch_bulk(args.atoms + at * kAtomBytes, static_cast<uint32_t>(n) * kAtomBytes);
      for (int kt = 0; kt < n; ++kt) {
        if (tile < args.tiles_n) l2_prefetch_bulk(args.tiles + (at + kt) * kLinearImageBytes, kLinearImageBytes);
        if (row < args.m) tma_prefetch_2d(&map_x, kt * 128, row);
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync_all();  // both CTAs' barriers exist before anything signals across the pair
  tc_fence_after();
  const uint32_t tmem_base = tmem_base_slot;
  // Every role waits for the launch in front itself, after what it can do before (its code comes into the instruction cache meanwhile).
  LinearArgs a = args;

  // The issuing warpgroup and the two epilogue warpgroups do not meet again before the kernel's last lines.
  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
    if (warp == 0) {
      // ---------------------------------------------------------------- code producer (both CTAs)
      pdl_wait();
      launder(a.tiles);
      if (cluster < total) scales_first_wait();
      if (lane == 0) {
        const uint32_t full0 = map_to_cta(smem_u32(&bar_full[0]), 0);  // the leader's barriers, as seen from this CTA
        uint32_t it = 0, s = 0, ph = 1u;
        bool ok = true;
        for (int u = cluster; u < total && ok; u += n_clusters) {
          units.at(u, pair, step);
          const int row = pair * 256 + static_cast<int>(rank) * 128;
          int rec = (2 * step + static_cast<int>(rank)) * tiles_k * 128;  // the images seen as rows of 128 bytes
          // Few clusters read a weight tile and wait for HBM with it: one of them asks for it ahead of the ring. (512 x 8192 -> 4096 29.7 -> 28.6
          // us, 777 x 6144 -> 6144 39.8 -> 38.9; with 16 that read it 4095 x 6144 -> 8192 150.7 -> 152.8.)
          const int ahead_end = units.pairs <= 4 && pair == 0 && 2 * step + static_cast<int>(rank) < a.tiles_n ? tiles_k - C::kAhead : 0;
          for (int kt = 0; kt < tiles_k; ++kt, ++it, rec += 128) {
            if (!mbar_wait(smem_u32(&bar_empty[s]), ph, abort_v, status)) { ok = false; break; }
            const uint32_t full = full0 + 8u * s, base = tiles + s * C::kStageBytes;
            if (leader) mbar_arrive_expect_tx(smem_u32(&bar_full[s]), 2 * C::kStageBytes);
            // rows beyond the last token or the last weight tile are read as zeros and count all the same
            tma_load_2d_pair(base, &map_x, kt * 128, row, full);
            tma_load_2d_pair(base + C::kWOff, &map_wc, 0, rec, full);
            if (kt < ahead_end)
              l2_prefetch_bulk(a.tiles + (static_cast<int64_t>(rec) + C::kAhead * 128) * 128, kLinearImageBytes);
            if (++s == C::kStages) { s = 0; ph ^= 1u; }
          }
        }
        if (!ok && leader) drain_copies(bar_full, it, C::kStages);
      }
    } else if (warp == 3) {
      // ---------------------------------------------------------------- scales (both CTAs): lane l writes 16 bytes of a token atom, rows l,
      // l + 32, l + 64 and l + 96. A group's bytes are asked for two groups ahead.
      const uint32_t sfull0 = map_to_cta(smem_u32(&bar_sfull[0]), 0);
      RowScales scales(a.scales, a.m, a.k);
      uint32_t even[4][5] = {}, odd[4][5] = {};
      int fu = cluster, fkt = 0;  // the group that is asked for next
      const auto fetch = [&](uint32_t (&v)[4][5]) {
        if (fu >= total) return;
        units.at(fu, pair, step);
        scales.load(static_cast<int64_t>(pair) * 256 + rank * 128 + lane, fkt, v);
        if ((fkt += kSfGroup) >= tiles_k) fkt = 0, fu += n_clusters;
      };
      uint32_t it = 0, slot = 0, ph = 1u;
      int u = cluster, kt = 0;  // the group that is stored next
      bool ok = true;
      const auto group = [&](uint32_t (&v)[4][5]) {
        if (u >= total || !ok) return;
        // free once its previous contents are in tensor memory
        if (!warp_wait(smem_u32(&bar_sf[slot]), ph, abort_v, status)) { ok = false; return; }
        const uint32_t sfull = sfull0 + 8u * slot, at = C::kSfOff + slot * C::kSfSlotBytes;
        units.at(u, pair, step);
        if (lane == 0) {
          const int atom = (2 * step * tiles_k + kt) * 4;  // the atoms seen as rows of 128 bytes
          if (leader) mbar_arrive_expect_tx(smem_u32(&bar_sfull[slot]), 4 * kSfGroup * kAtomBytes);
          // (a last group of fewer K-tiles brings the next tile's atoms or zeros along, which nothing reads)
          tma_load_2d_pair(tiles + at + kSfGroup * kAtomBytes, &map_ws, 0, atom, sfull);
          tma_load_2d_pair(tiles + at + 2 * kSfGroup * kAtomBytes, &map_ws, 0, atom + tiles_k * 4, sfull);
        }
        ++it;
        scales.tiles(static_cast<int64_t>(pair) * 256 + rank * 128 + lane, kt, v);
        uint4* cells = reinterpret_cast<uint4*>(tiles_ptr + at) + lane;
#pragma unroll
        for (int d = 0; d < kSfGroup; ++d) cells[d * 32] = make_uint4(v[0][d], v[1][d], v[2][d], v[3][d]);
        fence_proxy_async();
        __syncwarp();
        if (lane == 0) mbar_arrive(leader ? smem_u32(&bar_sfull[slot]) : smem_u32(&bar_relay[slot]));
        fetch(v);
        if ((kt += kSfGroup) >= tiles_k) kt = 0, u += n_clusters;
        if (++slot == C::kSfSlots) { slot = 0; ph ^= 1u; }
      };
      pdl_wait();
      launder(scales.base);
      fetch(even);
      if (cluster < total) scales_first_arrive();
      fetch(odd);
      while (u < total && ok) {
        group(even);
        group(odd);
      }
      if (!ok && leader && lane == 0) drain_copies(bar_sfull, it, C::kSfSlots);
    } else if (warp == 1) {
      // ---------------------------------------------------------------- MMA issue (leader only)
      if (leader) {
        // E4M3 x E4M3, UE8M0 scales, M = 256, N = 256; scale byte k of a row's cell for MMA k
        constexpr uint32_t kIdesc = (static_cast<uint32_t>(256 >> 3) << 17) | (1u << 23) | (static_cast<uint32_t>(256 >> 4) << 24);
        uint32_t ui = 0, s = 0, ph = 0, slot = 0, sph = 0, set = 0;
        bool ok = true, ready = false;
        pdl_wait();
        for (int u = cluster; u < total && ok; u += n_clusters, ++ui) {
          if (!warp_wait(smem_u32(&bar_tempty), (ui & 1u) ^ 1u, abort_v, status)) break;
          tc_fence_after();
          for (int kt = 0; kt < tiles_k && ok; kt += kSfGroup) {
            if (!warp_wait(smem_u32(&bar_sf[slot]), sph, abort_v, status)) { ok = false; break; }
            if (++slot == C::kSfSlots) { slot = 0; sph ^= 1u; }
            const int n = tiles_k - kt < kSfGroup ? tiles_k - kt : kSfGroup;
            uint32_t t_sft = tmem_base + C::kSfCol + set * kSfGroup * 16;
#pragma unroll 1
            for (int d = 0; d < n; ++d, t_sft += 16) {
              if (!__all_sync(0xffffffffu, ready || mbar_wait(smem_u32(&bar_full[s]), ph, abort_v, status))) { ok = false; break; }
              tc_fence_after();
              const uint32_t x_lo = (tiles + s * C::kStageBytes) >> 4, w_lo = x_lo + (C::kWOff >> 4), empty = smem_u32(&bar_empty[s]);
              const uint32_t t_sfw = t_sft + 8u;
              if (++s == C::kStages) { s = 0; ph ^= 1u; }
              ready = mbar_test(smem_u32(&bar_full[s]), ph);
              if (elect_one()) {
                tc_mma_mxf8_two(tmem_base, x_lo, w_lo, kIdesc, t_sft, t_sfw, static_cast<uint32_t>(kt + d != 0));
                tc_mma_mxf8_two(tmem_base, x_lo + 2, w_lo + 2, kIdesc | (1u << 29) | (1u << 4), t_sft, t_sfw, 1u);
                tc_mma_mxf8_two(tmem_base, x_lo + 4, w_lo + 4, kIdesc | (2u << 29) | (2u << 4), t_sft, t_sfw, 1u);
                tc_mma_mxf8_two(tmem_base, x_lo + 6, w_lo + 6, kIdesc | (3u << 29) | (3u << 4), t_sft, t_sfw, 1u);
                tc_commit_both(empty);  // the stage is free again, in both CTAs
                if (d == n - 1) tc_commit_pair(smem_u32(&bar_set[set]));
              }
              __syncwarp();
            }
            if (++set == kSfSets) set = 0;
          }
          if (ok && elect_one()) tc_commit_both(smem_u32(&bar_tfull));
        }
        if (__any_sync(0xffffffffu, *abort_v != 0) && elect_one()) drain_tcgen05_pair(smem_u32(&bar_drain[0]));
      }
    } else {
      // ---------------------------------------------------------------- scale copies into both CTAs' tensor memory (leader)
      if (leader) {
        uint32_t slot = 0, ph = 0, set = 0, set_ph = 1u;
        bool ok = true;
        pdl_wait();
        for (int u = cluster; u < total && ok; u += n_clusters) {
          for (int kt = 0; kt < tiles_k; kt += kSfGroup) {
            if (!__all_sync(0xffffffffu, mbar_wait_acquire_cluster(smem_u32(&bar_sfull[slot]), ph, abort_v, status) &&
                                             mbar_wait(smem_u32(&bar_set[set]), set_ph, abort_v, status))) {
              ok = false;
              break;
            }
            tc_fence_after();
            const int n = tiles_k - kt < kSfGroup ? tiles_k - kt : kSfGroup;
            const uint32_t lo = (tiles + C::kSfOff + slot * C::kSfSlotBytes) >> 4;
            const uint32_t t_sft = tmem_base + C::kSfCol + set * kSfGroup * 16, t_sfw = t_sft + 8u;
            if (elect_one()) {
              for (int d = 0; d < n; ++d) {
                const uint32_t from = lo + d * (kAtomBytes >> 4);
                tc_cp_scales_pair(t_sft + 16 * d, from);                                         // each CTA its own token rows
                tc_cp_scales_pair(t_sfw + 16 * d, from + (kSfGroup * kAtomBytes >> 4));          // weight rows 0..127 of N
                tc_cp_scales_pair(t_sfw + 16 * d + 4, from + (2 * kSfGroup * kAtomBytes >> 4));  // 128..255
              }
              tc_commit_both(smem_u32(&bar_sf[slot]));
            }
            __syncwarp();
            if (++slot == C::kSfSlots) { slot = 0; ph ^= 1u; }
            if (++set == kSfSets) { set = 0; set_ph ^= 1u; }
          }
        }
        if (__any_sync(0xffffffffu, *abort_v != 0) && elect_one()) drain_tcgen05_pair(smem_u32(&bar_drain[1]));
      } else if (lane == 0) {
        // -------------------------------------------------------------- the partner's token atoms are told to the leader
        const uint32_t sfull0 = map_to_cta(smem_u32(&bar_sfull[0]), 0);
        uint32_t slot = 0, ph = 0;
        bool ok = true;
        pdl_wait();
        for (int u = cluster; u < total && ok; u += n_clusters) {
          for (int kt = 0; kt < tiles_k; kt += kSfGroup) {
            if (!mbar_wait(smem_u32(&bar_relay[slot]), ph, abort_v, status)) { ok = false; break; }
            mbar_arrive_release_cluster(sfull0 + 8u * slot);
            if (++slot == C::kSfSlots) { slot = 0; ph ^= 1u; }
          }
        }
      }
    }
  } else {
    // ---------------------------------------------------------------- epilogue (both CTAs, warps 4..11)
    asm volatile("setmaxnreg.inc.sync.aligned.u32 208;");
    constexpr int kParts = 4;                                   // accumulator pieces of 32 columns
    constexpr int kOuts = KIND == kGated ? kParts / 2 : kParts; // pieces of 32 output columns
    const int q = warp & 3;                  // the TMEM lane quarter this warp may read
    const int half = (warp >> 2) - 1;        // which half of the unit's columns
    const uint32_t tempty_leader = map_to_cta(smem_u32(&bar_tempty), 0);
    float* const bias = reinterpret_cast<float*>(tiles_ptr + C::kBiasOff) + (warp - 4) * 128;
    const bool wide = (reinterpret_cast<uintptr_t>(a.out_codes) & 31) == 0;
    const bool scale_words = (a.n & 127) == 0 && (reinterpret_cast<uintptr_t>(a.out_scales) & 3) == 0;
    // the residual of piece i of a unit is in part i & 1 of the strip, the result in part 2
    const uint32_t strip = tiles + C::kStripOff + (warp - 4) * C::kStripBytes;
    uint8_t* const strip_row = tiles_ptr + C::kStripOff + (warp - 4) * C::kStripBytes + lane * 64;
    const uint32_t turn = (lane >> 1) & 3;                                     // the swizzle of a row's four 16-byte chunks
    const uint32_t res_bar = smem_u32(&bar_res[warp - 4][0]);
    const bool residual = a.residual != nullptr;
    // first token row and first output column of this warp's part of a unit
    const auto place = [&](int v, int64_t& row, int& col) {
      units.at(v, pair, step);
      row = static_cast<int64_t>(pair) * 256 + rank * 128 + q * 32;
      col = (2 * step + half) * (KIND == kGated ? 64 : 128);
    };
    // The residual of a piece (rows and columns beyond the matrix arrive as zeros); lane 0, once that part has been read.
    const auto ask_residual = [&](int64_t row, int col, int part) {
      mbar_arrive_expect_tx(res_bar + 8u * part, C::kPieceBytes);
      tma_load_2d(strip + part * C::kPieceBytes, &map_res, col, static_cast<int>(row), res_bar + 8u * part);
    };
    uint32_t ui = 0, res_ph = 0;  // res_ph: the phases of both parts (bit 0, bit 1)
    int64_t row0;
    int col0;
    int asked = 0;                // pieces asked for and not yet waited for
    pdl_wait();
    launder(a.bias);
    if (residual && cluster < total) {
      place(cluster, row0, col0);
      if (lane == 0) {
        ask_residual(row0, col0, 0);
        ask_residual(row0, col0 + 32, 1);
      }
      asked = 2;
    }
    for (int u = cluster; u < total; u += n_clusters, ++ui) {
      place(u, row0, col0);
      const int64_t row = row0 + lane;
      const bool in_row = row < a.m;
      // the bias in the order of the accumulator's columns
#pragma unroll
      for (int i = 0; i < kParts; ++i) {
        const int col = col0 + 32 * (KIND == kGated ? i >> 1 : i) + lane;
        const int64_t from = KIND == kGated && (i & 1) ? static_cast<int64_t>(a.n) + col : col;
        bias[32 * i + lane] = a.bias != nullptr && col < a.n ? __ldcg(a.bias + from) : 0.0f;
      }
      __syncwarp();
      // the warp decides together: tcgen05.ld below needs all 32 lanes
      if (!__all_sync(0xffffffffu, mbar_wait(smem_u32(&bar_tfull), ui & 1u, abort_v, status))) break;
      tc_fence_after();
      const uint32_t t_acc = tmem_base + 128 * half + (static_cast<uint32_t>(q * 32) << 16);
      uint32_t acc[kParts][32];
#pragma unroll
      for (int i = 0; i < kParts; ++i) tc_ld32_nowait(t_acc + 32 * i, acc[i]);
      asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive_cluster(tempty_leader);
      // A loop of one piece: unrolled, the code of a unit does not stay in the instruction cache. The piece is picked from the accumulator's
      // registers, or they move up behind it (GELU, gated); an activation takes 16 columns at a time, GELU 4. 2048 x 800 -> 5984: SiLU 26.2 us
      // (19 % more with the registers moving up and pair behind pair), GELU 27.8 (4 % more picked and 16 columns at a time).
      uint32_t scale_bytes = 0;
      bool ok = true;
#pragma unroll 1
      for (int i = 0; i < kOuts; ++i) {
        const int col = col0 + 32 * i;
        F2 y[16];
        const float* b_at = bias + 32 * (KIND == kGated ? 2 * i : i);
        constexpr int kTake = KIND == kLinear ? 16 : KIND == kGelu ? 2 : 8;  // pairs of columns at a time
        if (KIND == kGated) {
#pragma unroll
          for (int g = 0; g < 16; g += kTake) {
            constexpr int kUp = KIND == kGated ? 1 : 0;
            F2 gate[kTake], up[kTake];
#pragma unroll
            for (int k = 0; k < kTake; k += 2) {
              const float4 b = *reinterpret_cast<const float4*>(b_at + 2 * (g + k)), bu = *reinterpret_cast<const float4*>(b_at + 32 + 2 * (g + k));
              const int c = 2 * (g + k);
              gate[k] = F2{__uint_as_float(acc[0][c]), __uint_as_float(acc[0][c + 1])} + F2{b.x, b.y};
              gate[k + 1] = F2{__uint_as_float(acc[0][c + 2]), __uint_as_float(acc[0][c + 3])} + F2{b.z, b.w};
              up[k] = F2{__uint_as_float(acc[kUp][c]), __uint_as_float(acc[kUp][c + 1])} + F2{bu.x, bu.y};
              up[k + 1] = F2{__uint_as_float(acc[kUp][c + 2]), __uint_as_float(acc[kUp][c + 3])} + F2{bu.z, bu.w};
            }
            act_gated(gate, up, a.act);
#pragma unroll
            for (int k = 0; k < kTake; ++k) y[g + k] = gate[k];
          }
          if (i == 0) {
#pragma unroll
            for (int k = 0; k < 32; ++k) acc[0][k] = acc[2][k], acc[1][k] = acc[3][k];
          }
        } else {
          const auto pick = [&](const uint32_t (&from)[32]) {
#pragma unroll
            for (int k = 0; k < 16; ++k) y[k] = F2{__uint_as_float(from[2 * k]), __uint_as_float(from[2 * k + 1])};
          };
          if (KIND == kGelu || i == 0) pick(acc[0]);
          else if (i == 1) pick(acc[1]);
          else if (i == 2) pick(acc[2]);
          else pick(acc[3]);
#pragma unroll
          for (int g = 0; g < 16; g += kTake) {
            F2 r[kTake];
#pragma unroll
            for (int k = 0; k < kTake; k += 2) {
              const float4 b = *reinterpret_cast<const float4*>(b_at + 2 * (g + k));
              r[k] = y[g + k] + F2{b.x, b.y};
              r[k + 1] = y[g + k + 1] + F2{b.z, b.w};
            }
            act_of<KIND>(r, a.act);
#pragma unroll
            for (int k = 0; k < kTake; ++k) y[g + k] = r[k];
          }
        }
        if (KIND == kGelu) {
#pragma unroll
          for (int j = 0; j < 3; ++j)
#pragma unroll
            for (int k = 0; k < 32; ++k) acc[j][k] = acc[j + 1][k];
        }
        if (residual) {
          ok = __all_sync(0xffffffffu, mbar_wait(res_bar + 8u * (i & 1), (res_ph >> (i & 1)) & 1u, abort_v, status));
          if (!ok) break;
          res_ph ^= 1u << (i & 1);
          --asked;
#pragma unroll
          for (int p = 0; p < 4; ++p) {
            const uint4 r = *reinterpret_cast<const uint4*>(strip_row + (i & 1) * C::kPieceBytes + ((p ^ turn) << 4));
            const uint32_t rr[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
            for (int k = 0; k < 4; ++k)
              y[4 * p + k] = y[4 * p + k] + F2{__uint_as_float(rr[k] << 16), __uint_as_float(rr[k] & 0xffff0000u)};
          }
          // piece i + 2 goes where piece i was
          const bool here = i + 2 < kOuts;
          if (here || u + n_clusters < total) {
            int64_t next_row = row0;
            int next_col = col + 64;
            if (!here) {
              place(u + n_clusters, next_row, next_col);
              next_col += 32 * (i + 2 - kOuts);
            }
            __syncwarp();
            if (lane == 0) ask_residual(next_row, next_col, i & 1);
            ++asked;
          }
        }
        if (!MX) {  // the piece before has left
          if (lane == 0) tma_store_wait_read();
          __syncwarp();
        }
        if (MX) {
          float amax = 0.0f;
#pragma unroll
          for (int k = 0; k < 16; ++k) amax = max3_abs(amax, y[k].x, y[k].y);
          const int e = linear_scale(amax);
          const F2 inv = f2_dup(e8m0_value(static_cast<uint32_t>(254 - e)));
          uint32_t w[8];
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            const F2 lo = y[2 * k] * inv, hi = y[2 * k + 1] * inv;
            w[k] = pack_e4m3x4(lo.x, lo.y, hi.x, hi.y);
          }
          if (in_row && col < a.n) {  // (n is a multiple of 32 here)
            uint8_t* o = a.out_codes + row * a.n + col;
            if (wide) {
              st_sector(o, w);
            } else {
              reinterpret_cast<uint4*>(o)[0] = make_uint4(w[0], w[1], w[2], w[3]);
              reinterpret_cast<uint4*>(o)[1] = make_uint4(w[4], w[5], w[6], w[7]);
            }
            // four scales of a row are one store where they are one aligned word
            if (!scale_words || kOuts < 4) {
              a.out_scales[row * (a.n / 32) + col / 32] = static_cast<uint8_t>(e);
            } else {
              scale_bytes |= static_cast<uint32_t>(e) << (8 * i);
              if (i == 3) *reinterpret_cast<uint32_t*>(a.out_scales + row * (a.n / 32) + col / 32 - 3) = scale_bytes;
            }
          }
        } else {
#pragma unroll
          for (int p = 0; p < 4; ++p)
            *reinterpret_cast<uint4*>(strip_row + 2 * C::kPieceBytes + ((p ^ turn) << 4)) =
                make_uint4(pack_bf16x2(y[4 * p].x, y[4 * p].y), pack_bf16x2(y[4 * p + 1].x, y[4 * p + 1].y),
                           pack_bf16x2(y[4 * p + 2].x, y[4 * p + 2].y), pack_bf16x2(y[4 * p + 3].x, y[4 * p + 3].y));
        }
        if (!MX) {
          fence_proxy_async();
          __syncwarp();
          // (what lies beyond the matrix is not written)
          if (lane == 0 && row0 < a.m && col < a.n) tma_store_2d(&map_out, col, static_cast<int>(row0), strip + 2 * C::kPieceBytes);
        }
      }
      if (!ok) break;
      __syncwarp();  // all lanes have read this unit's bias
    }
    if (lane == 0) {
      if (!MX) tma_store_wait_read();
      if (asked > 0) {  // after an abort: the copies land before the CTA gives up its shared memory
        const uint64_t t0 = global_timer(), limit = wait_limit_ns();
        for (int h = 0; h < 2; ++h)
          while (!mbar_try_wait(res_bar + 8u * h, (res_ph >> h) & 1u) && global_timer() - t0 < limit) {}
      }
    }
  }

  tc_fence_before();
  __syncthreads();
  // Neither CTA frees tensor memory or leaves while the partner may still signal or read it. (Relaxed: a release would wait for the stores.)
  asm volatile("barrier.cluster.arrive.relaxed.aligned;\nbarrier.cluster.wait.aligned;" ::: "memory");
  if (warp == 1) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem_base),
                 "r"(static_cast<uint32_t>(C::kTmemCols))
                 : "memory");
  }
}

// ------------------------------------------------------------------------------------------------ host side
// bf16 rows [m][n], `stride` elements apart, boxes of 32 columns x 32 rows, 64-byte swizzle; columns and rows beyond are zeros / unwritten
static int make_rows_map(CUtensorMap* map, const void* base, int64_t n, int64_t m, int64_t stride) {
  EncodeTiledFn fn = encode_fn();
  if (!fn) return B200MOE_E_DRIVER;
  const cuuint64_t dims[2] = {static_cast<cuuint64_t>(n), static_cast<cuuint64_t>(m)};
  const cuuint64_t strides[1] = {static_cast<cuuint64_t>(m > 1 ? stride : n) * 2};
  const cuuint32_t box[2] = {32, 32}, estr[2] = {1, 1};
  const CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, const_cast<void*>(base), dims, strides, box, estr,
                        CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_64B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B,
                        CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? 0 : B200MOE_E_DRIVER;
}

template <int KIND, bool MX>
static int linear_pairs() {
  static PerDeviceAnswer<int> count;
  return resident_pairs_of(linear_pair_kernel<KIND, MX>, LinearPairCfg::kThreads, LinearPairCfg::kSmemBytes, count);
}

template <int KIND, bool MX>
static int launch_linear_pair(const LinearArgs& a, int32_t* status, cudaStream_t stream) {
  using C = LinearPairCfg;
  CUtensorMap mx, mwc, mws, mres = {}, mout = {};
  const uint64_t n_tiles = static_cast<uint64_t>(a.tiles_n) * a.tiles_k;
  int r;
  if ((r = make_map(&mx, a.codes, static_cast<uint64_t>(a.k), static_cast<uint64_t>(a.m), 128))) return r;
  if ((r = make_flat_map(&mwc, a.tiles, n_tiles * 128, 128))) return r;
  if ((r = make_flat_map(&mws, a.atoms, n_tiles * 4, kSfGroup * 4))) return r;
  if (a.residual && (r = make_rows_map(&mres, a.residual, a.n, a.m, a.residual_stride))) return r;
  if (a.out && (r = make_rows_map(&mout, a.out, a.n, a.m, a.out_stride))) return r;
  const int64_t units = (a.m + 255) / 256 * ((a.tiles_n + 1) / 2);
  if (units > 0x7fffffff) return B200MOE_E_ARG;
  const int pairs = linear_pairs<KIND, MX>();
  if (pairs <= 0) return B200MOE_E_DRIVER;
  return launch_pairs(linear_pair_kernel<KIND, MX>, units < pairs ? static_cast<int>(units) : pairs, C::kThreads, C::kSmemBytes, stream,
                      mx, mwc, mws, mres, mout, a, status);
}

template <int KIND>
static int linear_pair_out(const LinearArgs& a, int32_t* status, cudaStream_t stream) {
  return a.out ? launch_linear_pair<KIND, false>(a, status, stream) : launch_linear_pair<KIND, true>(a, status, stream);
}

int linear_pair(const LinearArgs& a, int32_t* status, cudaStream_t stream) {
  switch (a.act.kind) {
    case kLinear: return linear_pair_out<kLinear>(a, status, stream);
    case kSigmoid: return linear_pair_out<kSigmoid>(a, status, stream);
    case kGelu: return linear_pair_out<kGelu>(a, status, stream);
  }
  return linear_pair_out<kGated>(a, status, stream);
}

// Pairs of the call's kernel that are resident at once (0: cluster launch unavailable)
int linear_pair_resident(const LinearArgs& a) {
  switch (a.act.kind) {
    case kLinear: return a.out ? linear_pairs<kLinear, false>() : linear_pairs<kLinear, true>();
    case kSigmoid: return a.out ? linear_pairs<kSigmoid, false>() : linear_pairs<kSigmoid, true>();
    case kGelu: return a.out ? linear_pairs<kGelu, false>() : linear_pairs<kGelu, true>();
  }
  return a.out ? linear_pairs<kGated, false>() : linear_pairs<kGated, true>();
}

int set_wait_limit_linear_pair(unsigned long long ns) { return set_wait_limit_here(ns); }

}  // namespace b200moe
