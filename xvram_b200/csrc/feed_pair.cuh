// feed_pair.cuh -- the persistent CTA-pair kernel of the feed-forward operators, for more than
// 128 rows (operands, epilogues and the accumulators' columns: feed_common.cuh).
//
// A cluster of two CTAs computes accumulators of 256 rows x 256 columns (tcgen05
// cta_group::2): each CTA holds 128 rows of A and one of the two 128-row parts of B.
//
//   16-bit, HALVES = 1  a tile is 256 rows; two accumulators fill TMEM and alternate, so the
//               epilogue of a tile runs under the next tile's MMAs;
//   16-bit, HALVES = 2  a tile is 512 rows, 256 per CTA, both accumulators over the same B: a
//               quarter less operand traffic per FLOP.  The MMAs wait for the epilogues, which
//               run side by side; the next tile's first stages run on accumulator 0 alone
//               (kAhead stages) before accumulator 1 is needed;
//   MXFP4       a tile is 256 rows with one accumulator, emptied into registers first; the
//               other TMEM columns hold the stages' scales (each CTA's own A rows, all B rows).
//
//   warp 0      one lane per CTA: TMA loads into the stage ring, completion on the leader's
//               barrier;
//   warp 1      leader: one lane issues the MMAs and commits stages and accumulators to both CTAs;
//   warps 2..   epilogue per CTA, 8 warps per accumulator: two per TMEM lane quarter, splitting
//               the columns; their arrivals on the leader's barrier hand the accumulator back.
#pragma once

#include "feed_common.cuh"

namespace xvram::feed {

constexpr int kAhead = 3;
template <Kind K, int HALVES>
struct PairShape {
  static constexpr int kStages = K == Kind::mxf4 ? 5 : 4;
  static constexpr int kSlots = K == Kind::mxf4 ? 1 : 2; // accumulators
  static constexpr uint32_t kScales = (HALVES + 1) * kPart; // offset of a stage's scales
  static constexpr uint32_t kStage = kScales + (K == Kind::mxf4 ? kScaleBytes : 0);
  // 16-bit: two groups of 8 epilogue warps, a group per accumulator; MXFP4: one.
  static constexpr int kGroups = kSlots;
  static constexpr int kThreads = 64 + 256 * kGroups;
  static constexpr int kSmem = kStages * kStage + 8 * kStageBlock + 1024 + 256;
};

// The tile's batch and first row and column.  Tiles run in groups of 8 row tiles, so the
// pairs that work at the same time share both operands' tiles in L2.
__device__ __forceinline__ void tile_origin(const Params& p, int t, int rows, int cols, int& batch,
                                            int& m0, int& n0) {
  const int per_batch = p.tiles_m * p.tiles_n;
  batch = t / per_batch;
  const int tile = t % per_batch;
  const int span = 8 * p.tiles_n, first_m = (tile / span) * 8;
  const int group_m = min(8, p.tiles_m - first_m);
  m0 = (first_m + (tile % span) % group_m) * rows;
  n0 = ((tile % span) / group_m) * cols;
}

template <Kind K, Epilogue E, class T, int HALVES>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(PairShape<K, HALVES>::kThreads, 1)
    feed_pair_kernel(const __grid_constant__ Maps maps, const Params p) {
  constexpr int kTileN = E == Epilogue::gated ? 128 : 256;
  using Shape = PairShape<K, HALVES>;
  constexpr int kPairStages = Shape::kStages, kSlots = Shape::kSlots;
  constexpr uint32_t kStage = Shape::kStage;
  constexpr int kElems = K == Kind::f16 ? 64 : 128; // map elements per 128-byte row
  extern __shared__ unsigned char smem_raw[];
  unsigned char* smem = reinterpret_cast<unsigned char*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  unsigned char* blocks = smem + kPairStages * kStage;
  uint64_t* full = reinterpret_cast<uint64_t*>(blocks + 8 * kStageBlock);
  uint64_t* empty = full + kPairStages;
  uint64_t* acc_full = empty + kPairStages; // [2]
  uint64_t* acc_empty = acc_full + 2;       // [2]
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acc_empty + 2);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const uint32_t rank = tc::cluster_rank();
  const int pairs = gridDim.x >> 1, first = blockIdx.x >> 1;
  const int tiles = p.batches * p.tiles_m * p.tiles_n;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (tid == 0) {
    for (int s = 0; s < kPairStages; ++s) {
      mbar_init(&full[s], 1); // used on the leader
      mbar_init(&empty[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&acc_full[b], 1);
      mbar_init(&acc_empty[b], 16); // used on the leader: 8 epilogue warps of both CTAs
    }
    *abort_flag = 0;
    fence_mbarrier_init();
  }
  if (warp == 1)
    tc::tmem_alloc<2>(tmem_slot, kTmemCols);
  tc::fence_before();
  tc::cluster_sync(); // both CTAs' barriers exist before any cross-CTA arrival
  tc::fence_after();
  const uint32_t tmem = *tmem_slot;
  const uint32_t sbase = smem_u32(smem);

  if (warp == 0) {
    // ---------------------------------------------------------------- producer
    if (lane == 0) {
      int s = 0;          // stage, and the parity of its last release
      uint32_t phase = 1; // (a fresh barrier's previous phase: the first round does not wait)
      long long issued = 0;
      bool stop = false;
      for (int t = first; t < tiles && !stop; t += pairs) {
        int batch, m0, n0;
        tile_origin(p, t, 256 * HALVES, kTileN, batch, m0, n0);
        m0 += 128 * HALVES * static_cast<int>(rank);
        const int row = E == Epilogue::gated ? n0 : n0 + 128 * static_cast<int>(rank);
        for (int kt = 0; kt < p.k_tiles; ++kt) {
          if (*abort_flag || !mbar_wait_bounded(&empty[s], phase, p.timeout_ns)) {
            atomicOr(&feed_error, 2u);
            *abort_flag = 1;
            stop = true;
            break;
          }
          const int seg = kt >= p.k_split;
          const CUtensorMap* ma = &maps.a[seg | batch];
          const CUtensorMap* mb = &maps.b[E == Epilogue::gated ? rank : seg];
          const int k0 = (kt - (seg ? p.k_split : 0)) * kElems;
          const uint32_t bar = tc::cluster_addr(smem_u32(&full[s]), 0);
          const uint32_t a = sbase + s * kStage, b = a + HALVES * kPart;
          if (rank == 0)
            mbar_arrive_expect_tx(&full[s], 2 * kStage); // both CTAs' copies
#pragma unroll
          for (int i = 0; i < HALVES; ++i) {
            if (K == Kind::f16 && p.a_mn) {
              tc::tma_load<2>(a + i * kPart, ma, bar, m0 + 128 * i, k0);
              tc::tma_load<2>(a + i * kPart + kPart / 2, ma, bar, m0 + 128 * i + 64, k0);
            } else {
              tc::tma_load<2>(a + i * kPart, ma, bar, k0, m0 + 128 * i);
            }
          }
          if (K == Kind::f16 && p.b_mn) {
            tc::tma_load<2>(b, mb, bar, row, k0);
            tc::tma_load<2>(b + kPart / 2, mb, bar, row + 64, k0);
          } else {
            tc::tma_load<2>(b, mb, bar, k0, row);
          }
          if constexpr (K == Kind::mxf4) {
            const uint32_t sc = sbase + s * kStage + Shape::kScales;
            tc::tma_load<2>(sc, &maps.scale_a, bar, kt * 256, m0 / 128);
#pragma unroll
            for (int j = 0; j < 2; ++j)
              tc::tma_load<2>(sc + kScaleTile * (1 + j),
                              &maps.scale_b[E == Epilogue::gated ? j : 0], bar, kt * 256,
                              E == Epilogue::gated ? n0 / 128 : n0 / 128 + j);
          }
          ++issued;
          if (++s == kPairStages) {
            s = 0;
            phase ^= 1;
          }
        }
      }
      // Drain: every stage filled here has been consumed (or times out) before exit.
      for (long long i = issued > kPairStages ? issued - kPairStages : 0; i < issued; ++i) {
        if (!mbar_wait_bounded(&empty[i % kPairStages], (i / kPairStages) & 1, p.timeout_ns)) {
          atomicOr(&feed_error, 4u);
          break;
        }
      }
    }
  } else if (warp == 1) {
    // ------------------------------------------------- MMA issuer (pair leader)
    if (rank == 0 && lane == 0) {
      const uint32_t sempty = smem_u32(empty), sacc = smem_u32(acc_full);
      int s = 0;
      uint32_t phase = 0;
      int units = 0; // accumulators used so far
      const auto fail = [&] {
        atomicOr(&feed_error, 1u);
        *abort_flag = 1;
      };
      const auto take = [&](int unit) { // accumulator unit % kSlots is free
        const int use = unit / kSlots;
        const bool ok = use == 0 || mbar_wait_bounded(&acc_empty[unit % kSlots], (use - 1) & 1,
                                                      p.timeout_ns);
        tc::fence_after();
        return ok;
      };
      const auto multiply = [&](int stage, int half, uint32_t d, bool first_k) {
        const uint32_t base = sbase + stage * kStage;
        const uint32_t a = base + half * kPart, b = base + HALVES * kPart;
        if constexpr (K == Kind::f16)
          stage_f16<2>(p, d, a, b, first_k);
        else
          stage_mxf4<2>(p, d, a, b, base + Shape::kScales, base + Shape::kScales + kScaleTile,
                        tmem + kScaleCol + stage * kScaleCols, first_k);
      };
      const auto next = [&] {
        if (++s == kPairStages) {
          s = 0;
          phase ^= 1;
        }
      };
      bool stop = false;
      for (int t = first; t < tiles && !stop; t += pairs, units += HALVES) {
        if (!take(units)) {
          fail();
          break;
        }
        const uint32_t d0 = tmem + 256 * (units % kSlots);
        int kt = 0;
        if constexpr (HALVES == 2) {
          // The first stages on accumulator 0 alone, then the same stages on accumulator 1.
          const int ahead = min(kAhead, p.k_tiles), s0 = s;
          for (; kt < ahead && !stop; ++kt) {
            if (*abort_flag || !mbar_wait_bounded(&full[s], phase, p.timeout_ns)) {
              stop = true;
              break;
            }
            tc::fence_after();
            multiply(s, 0, d0, kt == 0);
            next();
          }
          if (stop || !take(units + 1)) {
            fail();
            break;
          }
          for (int i = 0; i < ahead; ++i) {
            const int stage = s0 + i < kPairStages ? s0 + i : s0 + i - kPairStages;
            multiply(stage, 1, tmem + 256, i == 0);
            tc::mma_commit_both(sempty + 8 * stage);
          }
        }
        for (; kt < p.k_tiles; ++kt) {
          if (*abort_flag || !mbar_wait_bounded(&full[s], phase, p.timeout_ns)) {
            fail();
            stop = true;
            break;
          }
          tc::fence_after();
          multiply(s, 0, d0, kt == 0);
          if constexpr (HALVES == 2)
            multiply(s, 1, tmem + 256, false);
          tc::mma_commit_both(sempty + 8 * s);
          next();
        }
        if (!stop) {
          tc::mma_commit_both(sacc + 8 * (units % kSlots));
          if constexpr (HALVES == 2)
            tc::mma_commit_both(sacc + 8);
        }
      }
    }
    __syncwarp();
  } else {
    // ---------------------------------------------------------------- epilogue
    // Group g of 8 warps takes accumulator g's units; a unit is a tile's (half's) accumulator.
    const int quad = warp & 3, half = ((warp - 2) >> 2) & 1, group = (warp - 2) >> 3;
    const uint32_t release = tc::cluster_addr(smem_u32(acc_empty), 0) + 8 * group;
    int unit = 0;
    bool stop = false;
    float unscale = 1.0f;
    if constexpr (K == Kind::f16 && E == Epilogue::plain && std::is_same_v<T, __half>)
      unscale = fp16_unscale(p.top);
    for (int t = first; t < tiles && !stop; t += pairs) {
      int batch, m0, n0;
      tile_origin(p, t, 256 * HALVES, kTileN, batch, m0, n0);
      T* out = static_cast<T*>(p.out[batch]);
      for (int i = 0; i < HALVES; ++i, ++unit) {
        if (unit % Shape::kGroups != group)
          continue;
        const int row0 = m0 + 128 * (HALVES * static_cast<int>(rank) + i) + 32 * quad;
        const bool ok = mbar_wait_bounded(&acc_full[group], (unit / kSlots) & 1,
                                          p.timeout_ns * 4);
        if (!ok) {
          atomicOr(&feed_error, 8u);
          *abort_flag = 1;
        }
        tc::fence_after();
        if (!__all_sync(0xffffffffu, ok && !*abort_flag)) {
          stop = true;
          break;
        }
        const uint32_t t_row = tmem + 256 * group + (static_cast<uint32_t>(32 * quad) << 16);
        const auto hand_back = [&] {
          tc::fence_before();
          __syncwarp();
          if (lane == 0)
            tc::mbar_arrive_cluster(release);
        };
        const int col = n0 + half * (kTileN / 2);
        if constexpr (K == Kind::mxf4) {
          // One accumulator: emptied into registers, so that the next tile's MMAs wait only for that.
          float r[128];
          load_accumulator<E>(t_row, half, r);
          hand_back();
          finish_rows<E, T>(p, r, row0, col, out, blocks + (warp - 2) * kStageBlock);
        } else {
          finish_unit<E, T>(p, t_row, half, row0, col, out, blocks + (warp - 2) * kSubBlock,
                            unscale, hand_back);
        }
      }
    }
  }

  // Neither CTA leaves (or frees TMEM) while its partner may still use its shared memory
  // or TMEM: every wait above is bounded, so both CTAs reach this point.
  tc::fence_before();
  __syncthreads();
  tc::cluster_sync();
  if (warp == 1) {
    tc::fence_after();
    tc::tmem_free<2>(tmem, kTmemCols);
  }
}

template <Kind K, Epilogue E, class T, int HALVES>
cudaError_t launch_pairs(const Maps& maps, Params p, cudaStream_t stream) {
  static std::atomic<uint64_t> done{0};
  const auto kernel = feed_pair_kernel<K, E, T, HALVES>;
  constexpr int smem = PairShape<K, HALVES>::kSmem;
  static_assert(smem <= 232448, "shared memory of one CTA per SM");
  if (cudaError_t e = tc::allow_smem(kernel, smem, done); e != cudaSuccess)
    return e;
  p.tiles_m = (p.m + 256 * HALVES - 1) / (256 * HALVES);
  const long long tiles = static_cast<long long>(p.batches) * p.tiles_m * p.tiles_n;
  if (tiles <= 0 || tiles > 0x7fffffffll)
    return cudaErrorInvalidConfiguration;
  const int pairs = static_cast<int>(std::min<long long>(tiles, tc::sm_count() / 2));
  kernel<<<2 * pairs, PairShape<K, HALVES>::kThreads, smem, stream>>>(maps, p);
  return cudaGetLastError();
}

} // namespace xvram::feed
