// Product of two microscaled 4-bit matrices:  P[R, S] = X[R, K] * W[S, K]^T  with block scales on both
// operands, fp32 accumulation in tensor memory, 16-bit output.
//
//   P[r, s] = sum over blocks b of  sx[r, b] * sw[s, b] * sum over k in b of  x[r, k] * w[s, k]
//
// The tensor cores apply the scales themselves (tcgen05.mma.kind::mxf4 / mxf4nvf4): a K-tile of 256
// elements is 128 bytes of codes per row — the same swizzled rows as 64 16-bit elements — plus 1 KB
// (MXFP4) or 2 KB (NVFP4) of scales per 128 rows, stored so that one TMA box brings them in and
// tcgen05.cp moves them to tensor memory unchanged.
//
//   warp 0      TMA producer: codes and scales of both operands into a shared-memory ring
//   warp 1      MMA issuer: four MMAs of K = 64 per K-tile
//   warp 2      scale copies: shared -> tensor memory, ahead of the MMAs (issued by the MMA warp itself, 6 to 12 copies per
//               K-tile kept the tensor cores waiting: 8192^3 MXFP4 273 us, NVFP4 353 us, against 194 and 215)
//   warps 3-6   epilogue: accumulator -> registers -> C
//
// X's rows ride on the MMA's M (128 per CTA), W's on its N (BN per tile). PAIR = 1 drives two CTAs with one
// cta_group::2 MMA: 256 x BN, each CTA staging its own rows of X and half of W's. Feeding these
// MMAs is what limits a large product: a K-tile of a lone 128 x 256 tile takes 540 cycles at the nominal rate and
// 51 KB of loads, 94 bytes per cycle and SM; a pair loads 35 KB for the same work. Measured, 8192^3 MXFP4: 194 us in a
// burst (5.7 PFLOP/s) and 229 us for seconds, where the power limit holds the clock at 1.4 GHz; the loads
// alone take 140 us, the MMAs alone 122 us at the full clock. 16 x 28672 x 8192 NVFP4: 23.4 us, 5.7 TB/s.
//
// C is X W^T row-major (A is X), or its transpose (the weights are X: `transposed`). The transposed form
// serves few rows, so that no tensor work and no accumulator is spent on padding, and everything that
// is short of tiles: there a cluster of CTAs (pairs) shares one tile, each taking a range of K, and the
// partial tiles are added over distributed shared memory in rank order. No workspace is needed, nothing depends on
// timing and a captured launch can be replayed.
//
// Tensor memory (512 columns): two accumulators, and the scales of the last kScaleBuffers K-tiles. With
// BN = 256 the accumulators overlap by the columns the scales need: the epilogue reads those first and
// hands them back before the rest, so all the next tile waits for is that part of the read-out.
#pragma once

#include "desc.cuh"
#include "mx_format.cuh"
#include "ptx.cuh"
#include "scheduler.cuh"
#include "status.cuh"

namespace b200 {

struct MxGemmArgs {
  int R, S;            // rows of X and W
  int k_tiles;         // K-tiles of 256 elements
  SchedParams sched;   // whole tiles in raster order
  int split;           // CTAs (pairs) that share a tile; above 1 every cluster has one tile
  int stages;
  int transposed;      // 1: element (r, s) goes to C[s * ldc + r]
  int tma_store;       // 1: rows of C start on 16 bytes and S is a multiple of 8 (row-major only)
  int slab_bytes;      // epilogue staging per warp (row-major only)
  uint16_t* C;
  long long ldc;
  float alpha, beta;
  int scale;           // 1: C = acc * alpha + beta
  unsigned int* status;
};

static constexpr int kMxMaxStages = 16;
static constexpr int kMxSlabBytes = 32 * 64;  // 32 rows x 32 columns of 16-bit output
static constexpr int kMxSlabs = 2;            // per epilogue warp
// Rows of C that do not start on 16 bytes: a warp stages 32 rows of 128 columns (16 bytes of padding against bank
// conflicts) and writes them as aligned 16-byte pieces; element by element, the partial sectors cost
// 777 x 5003 x 4104 NVFP4 18 us of 36.
static constexpr int kMxRowCols = 128;
static constexpr int kMxRowPitch = 2 * kMxRowCols + 16;

template <int FMT, int BN, int PAIR>
struct MxGemmTraits {
  static constexpr int kThreads = 224;
  static constexpr int kCtas = PAIR ? 2 : 1;
  static constexpr int kTileRows = 128 * kCtas;
  static constexpr int kSBlocks = (BN + 127) / 128;                 // scale tiles of W per K-tile
  static constexpr int kXBytes = 128 * 128;
  static constexpr int kWRows = BN / kCtas;                         // staged by one CTA
  static constexpr int kWBytes = kWRows * 128;
  static constexpr int kScaleTile = mx_tile_bytes(FMT);
  static constexpr int kGroups = mx_tile_groups(FMT);
  static constexpr int kStageBytes = kXBytes + kWBytes + (1 + kSBlocks) * kScaleTile;
  static constexpr int kScaleCols = kGroups * 4 * (1 + kSBlocks);   // of one K-tile: X's, then W's
  // K-tiles whose scales tensor memory holds; never more than the ring has stages. Three where tensor memory or the ring
  // (BN = 256), or half an SM's shared memory (64, NVFP4) has no room for a fourth.
  static constexpr int kScaleBuffers = BN == 256 || (FMT == kNvfp4 && BN == 64) ? 3 : 4;
  static constexpr int kScalesNeed = kScaleBuffers * kScaleCols;
  static constexpr int kAccCols = BN < 32 ? 32 : BN;
  // Columns the two accumulators share, in whole 32-column reads.
  static constexpr int kOverlap = 2 * kAccCols + kScalesNeed > 512 ? (2 * kAccCols + kScalesNeed - 512 + 31) / 32 * 32 : 0;
  static constexpr int kAcc1 = kAccCols - kOverlap;                 // first column of the second accumulator
  static constexpr int kScales0 = kAcc1 + kAccCols;
  static constexpr int kNeedCols = kScales0 + kScalesNeed;
  static constexpr int kTmemCols = kNeedCols <= 128 ? 128 : kNeedCols <= 256 ? 256 : 512;
  static_assert(kNeedCols <= 512, "accumulators and scales exceed tensor memory");
  static_assert(BN % 16 == 0 && BN <= 256 && (!PAIR || BN >= 64), "width of the MMA");
  static_assert(kWBytes % 1024 == 0, "swizzled tiles start on 1024 bytes");
  // Row-major C comes from the widest tile alone; the narrower ones always write the transposed form.
  static constexpr bool kRowMajor = BN == 256;
  static constexpr int kBarrierBytes = 512;
  static constexpr int smem_bytes(int stages, int slabs) { return 1024 + stages * kStageBytes + 4 * slabs + kBarrierBytes; }
};

__device__ __forceinline__ void mx_report_timeout(unsigned int* status, unsigned int code, int tile, int detail,
                                                  volatile uint32_t* abort_flag) {
  if (atomicCAS(status, 0u, code) == 0u) {
    status[1] = blockIdx.x;
    status[2] = static_cast<unsigned int>(tile);
    status[3] = static_cast<unsigned int>(detail);
  }
  *abort_flag = 1u;
}

template <int F16>
__device__ __forceinline__ uint32_t mx_pack16(float lo, float hi) {
  uint32_t r;
  if constexpr (F16) {
    asm("cvt.rn.f16x2.f32 %0, %2, %1;" : "=r"(r) : "f"(lo), "f"(hi));
  } else {
    asm("cvt.rn.bf16x2.f32 %0, %2, %1;" : "=r"(r) : "f"(lo), "f"(hi));
  }
  return r;
}

__device__ __forceinline__ float mx_finish(const MxGemmArgs& args, float acc) {
  return args.scale ? __fadd_rn(__fmul_rn(acc, args.alpha), args.beta) : acc;
}

// A bounded wait of a whole warp: one answer for all lanes, so that the warp stays converged whichever lane's budget
// runs out first.
__device__ __forceinline__ bool mx_warp_wait(uint32_t bar, uint32_t parity) {
  return __all_sync(0xffffffffu, ptx::mbar_wait(bar, parity));
}

// Grid: clusters of split * (1 or 2) CTAs. Pair p of a cluster takes K-tiles
// [k_tiles * p / split, k_tiles * (p + 1) / split) of each of the cluster's tiles.
template <int FMT, int BN, int PAIR, int F16>
__global__ void __launch_bounds__(224) mx_gemm_kernel(const __grid_constant__ CUtensorMap map_x,
                                                       const __grid_constant__ CUtensorMap map_w,
                                                       const __grid_constant__ CUtensorMap map_sx,
                                                       const __grid_constant__ CUtensorMap map_sw,
                                                       const __grid_constant__ CUtensorMap map_c,
                                                       const __grid_constant__ MxGemmArgs args) {
  using T = MxGemmTraits<FMT, BN, PAIR>;
  constexpr int G = T::kCtas;
  extern __shared__ uint8_t smem_raw[];
  const int warp = __shfl_sync(0xffffffffu, static_cast<int>(threadIdx.x) / 32, 0);
  const uint32_t lane = ptx::lane_id();
  const int cluster_size = args.split * G;
  const int cluster = static_cast<int>(blockIdx.x) / cluster_size;
  const uint32_t cluster_rank = cluster_size > 1 ? ptx::cluster_ctarank() : 0u;
  const uint32_t cta = PAIR ? cluster_rank & 1u : 0u;  // of the pair
  const uint32_t leader = cluster_rank - cta;
  const int part = static_cast<int>(cluster_rank) / G;
  const int kt0 = static_cast<int>(static_cast<long long>(args.k_tiles) * part / args.split);
  const int kt1 = static_cast<int>(static_cast<long long>(args.k_tiles) * (part + 1) / args.split);

  const uint32_t smem_base = (ptx::smem_u32(smem_raw) + 1023u) & ~1023u;
  const uint32_t slab_base = smem_base + static_cast<uint32_t>(args.stages * T::kStageBytes);
  const uint32_t bar_base = slab_base + static_cast<uint32_t>(4 * args.slab_bytes);
  auto stage_addr = [&](int s) { return smem_base + static_cast<uint32_t>(s * T::kStageBytes); };
  auto full_bar = [&](int s) { return bar_base + 8u * static_cast<uint32_t>(s); };
  auto empty_bar = [&](int s) { return bar_base + 8u * static_cast<uint32_t>(kMxMaxStages + s); };
  auto done_bar = [&](int a) { return bar_base + 8u * static_cast<uint32_t>(2 * kMxMaxStages + a); };
  auto drained_bar = [&](int a) { return bar_base + 8u * static_cast<uint32_t>(2 * kMxMaxStages + 2 + a); };
  auto scales_bar = [&](int b) { return bar_base + 8u * static_cast<uint32_t>(2 * kMxMaxStages + 4 + b); };
  const uint32_t tmem_slot = bar_base + 8u * (2 * kMxMaxStages + 8);
  uint8_t* generic_bar = smem_raw + (bar_base - ptx::smem_u32(smem_raw));
  volatile uint32_t* tmem_ptr = reinterpret_cast<volatile uint32_t*>(generic_bar + 8 * (2 * kMxMaxStages + 8));
  volatile uint32_t* abort_flag = tmem_ptr + 1;

  if (warp == 0 && lane == 0) {
    ptx::prefetch_tensormap(&map_x);
    ptx::prefetch_tensormap(&map_w);
    ptx::prefetch_tensormap(&map_sx);
    ptx::prefetch_tensormap(&map_sw);
    if (T::kRowMajor && args.tma_store) ptx::prefetch_tensormap(&map_c);
    for (int s = 0; s < args.stages; ++s) {
      ptx::mbar_init(full_bar(s), 1);
      ptx::mbar_init(empty_bar(s), 1);
    }
    for (int a = 0; a < 2; ++a) {
      ptx::mbar_init(done_bar(a), 1);
      ptx::mbar_init(drained_bar(a), 4 * G);
    }
    for (int b = 0; b < T::kScaleBuffers; ++b) ptx::mbar_init(scales_bar(b), 1);
    *abort_flag = 0u;
    ptx::fence_mbar_init();
  }
  if (warp == 1) {
    ptx::tmem_alloc<G>(tmem_slot, T::kTmemCols);
    ptx::tmem_relinquish<G>();
  }
  ptx::tc_fence_before_sync();
  __syncthreads();
  if (PAIR) {
    ptx::cluster_arrive();
    ptx::cluster_wait();
  }
  ptx::tc_fence_after_sync();
  const uint32_t tmem_base = *tmem_ptr;
  ptx::grid_launch_dependents();  // (not before this CTA has its tensor memory: the next kernel's may wait for it)
  ptx::grid_dependency_wait();

  if (warp == 0) {
    if (lane == 0) {
      const uint32_t leader_full = PAIR ? ptx::map_to_cta(full_bar(0), leader) : full_bar(0);
      constexpr int kBoxes = T::kScaleTile / 1024;  // 1 KB rows of the scale maps per tile
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int tile = cluster; ok && tile < args.sched.num_tiles; tile += args.sched.num_workers) {
        const TileCoord tc = tile_coord(args.sched, tile);
        const int r0 = tc.m * T::kTileRows + static_cast<int>(cta) * 128;
        const int s0 = tc.n * BN;
        const int w0 = s0 + static_cast<int>(cta) * T::kWRows;
        const int sx_tile = (r0 / kMxTileRows) * args.k_tiles, sw_tile = (s0 / kMxTileRows) * args.k_tiles;
        for (int kt = kt0; kt < kt1; ++kt) {
          if (!ptx::mbar_wait(empty_bar(stage), phase ^ 1u)) {
            mx_report_timeout(args.status, kStatusProducerTimeout, tile, kt, abort_flag);
            ok = false;
            break;
          }
          const uint32_t full = leader_full + 8u * static_cast<uint32_t>(stage), x = stage_addr(stage);
          const uint32_t w = x + T::kXBytes, sx = w + T::kWBytes, sw = sx + T::kScaleTile;
          if (cta == 0) ptx::mbar_arrive_expect_tx(full_bar(stage), T::kStageBytes * G);
          auto load = [&](uint32_t dst, const CUtensorMap* map, int c0, int c1) {
            if (PAIR) {
              ptx::tma_load_3d_pair(dst, map, full, c0, c1, 0);
            } else {
              ptx::tma_load_3d(dst, map, full, c0, c1, 0);
            }
          };
          load(x, &map_x, kt * 128, r0);
          load(w, &map_w, kt * 128, w0);
          load(sx, &map_sx, 0, (sx_tile + kt) * kBoxes);
#pragma unroll
          for (int b = 0; b < T::kSBlocks; ++b) {
            load(sw + b * T::kScaleTile, &map_sw, 0, (sw_tile + b * args.k_tiles + kt) * kBoxes);
          }
          if (++stage == args.stages) {
            stage = 0;
            phase ^= 1u;
          }
        }
      }
    }
    __syncwarp();
  } else if (warp <= 2) {
    const uint16_t both = static_cast<uint16_t>(3u << leader);
    const int len = kt1 - kt0;
    const int mine = args.sched.num_tiles > cluster ? (args.sched.num_tiles - cluster - 1) / args.sched.num_workers + 1 : 0;
    if (warp == 1 && cta == 0) {
      // 16-element blocks: every MMA has a scale column of its own; 32-element blocks: two MMAs share
      // one, the second starting at its upper byte pair.
      constexpr uint32_t idesc0 = make_instr_desc_mxf4(T::kTileRows, BN, FMT == kMxfp4, 0);
      constexpr uint32_t idesc1 = make_instr_desc_mxf4(T::kTileRows, BN, FMT == kMxfp4, FMT == kMxfp4 ? 2 : 0);
      auto commit = [&](uint32_t bar) {
        if (PAIR) {
          ptx::umma_commit_pair(bar, both);
        } else {
          ptx::umma_commit_1cta(bar);
        }
      };
      // The whole warp runs the loop and one elected lane issues: with a single lane in the loop an issue costs more
      // (16 x 28672 x 8192 NVFP4 24.4 against 23.4 us, 1 x 4096 x 4096 5.7 against 5.2 us).
      const uint64_t desc0 = make_smem_desc_sw128(smem_base);
      uint64_t desc = desc0;
      int stage = 0, buffer = 0;
      uint32_t phase = 0, scales_phase = 0;
      bool ok = true;
      for (int turn = 0; ok && turn < mine; ++turn) {
        // Overlapping accumulators: the tile before must have been read out where they overlap.
        // Separate ones: the tile before that, entirely.
        const bool wait_drained = T::kOverlap > 0 ? turn >= 1 : turn >= 2;
        const uint32_t drained_phase = static_cast<uint32_t>(T::kOverlap > 0 ? turn - 1 : turn / 2 - 1) & 1u;
        if (wait_drained && !mx_warp_wait(drained_bar(T::kOverlap > 0 ? 0 : turn & 1), drained_phase)) {
          mx_report_timeout(args.status, kStatusMmaTmemTimeout, turn, 0, abort_flag);
          break;
        }
        const uint32_t tmem_d = tmem_base + ((turn & 1) ? T::kAcc1 : 0);
        for (int k_tile = 0; k_tile < len; ++k_tile) {
          // (the copies were issued after the stage had landed, so the second wait only orders this thread)
          if (!mx_warp_wait(scales_bar(buffer), scales_phase) || !mx_warp_wait(full_bar(stage), phase)) {
            mx_report_timeout(args.status, kStatusMmaFullTimeout, turn, k_tile, abort_flag);
            ok = false;
            break;
          }
          ptx::tc_fence_after_sync();
          const uint32_t tsx = tmem_base + T::kScales0 + static_cast<uint32_t>(buffer * T::kScaleCols);
          const uint32_t tsw = tsx + T::kGroups * 4;
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const int g = FMT == kMxfp4 ? k / 2 : k;
            if (ptx::elect_one()) {
              ptx::umma_mxf4<G, FMT == kNvfp4>(tmem_d, desc + k * kDescKStep, desc + (T::kXBytes >> 4) + k * kDescKStep,
                                               (k & 1) ? idesc1 : idesc0, tsx + g * 4, tsw + g * 4 * T::kSBlocks,
                                               (k_tile > 0 || k > 0) ? 1u : 0u);
            }
          }
          if (ptx::elect_one()) commit(empty_bar(stage));
          __syncwarp();
          desc += T::kStageBytes >> 4;
          if (++stage == args.stages) {
            stage = 0;
            phase ^= 1u;
            desc = desc0;
          }
          if (++buffer == T::kScaleBuffers) {
            buffer = 0;
            scales_phase ^= 1u;
          }
        }
        if (ok && ptx::elect_one()) commit(done_bar(turn & 1));
        __syncwarp();
      }
    } else if (warp == 2 && cta == 0) {
      const long long total = static_cast<long long>(mine) * len;  // K-tiles of all tiles, one sequence
      const uint64_t desc0 = make_smem_desc_scales(smem_base + T::kXBytes + T::kWBytes);
      uint64_t desc = desc0;
      int stage = 0, buffer = 0, old_stage = 0;
      uint32_t phase = 0, old_phase = 0;
      for (long long i = 0; i < total; ++i) {
        if (i >= T::kScaleBuffers) {
          // What the buffer holds, the scales of the K-tile kScaleBuffers before, must have been used.
          if (!mx_warp_wait(empty_bar(old_stage), old_phase)) {
            mx_report_timeout(args.status, kStatusMmaTmemTimeout, cluster, static_cast<int>(i), abort_flag);
            break;
          }
          if (++old_stage == args.stages) {
            old_stage = 0;
            old_phase ^= 1u;
          }
        }
        if (!mx_warp_wait(full_bar(stage), phase)) {
          mx_report_timeout(args.status, kStatusMmaFullTimeout, cluster, static_cast<int>(i), abort_flag);
          break;
        }
        ptx::tc_fence_after_sync();
        const uint32_t tsx = tmem_base + T::kScales0 + static_cast<uint32_t>(buffer * T::kScaleCols);
        const uint32_t tsw = tsx + T::kGroups * 4;
        if (ptx::elect_one()) {
#pragma unroll
          for (int g = 0; g < T::kGroups; ++g) {
            ptx::tmem_copy_scales<G>(tsx + g * 4, desc + g * (kMxGroupBytes >> 4));
#pragma unroll
            for (int b = 0; b < T::kSBlocks; ++b) {
              ptx::tmem_copy_scales<G>(tsw + (g * T::kSBlocks + b) * 4,
                                       desc + ((b + 1) * T::kScaleTile + g * kMxGroupBytes) / 16);
            }
          }
          if (PAIR) {
            ptx::umma_commit_pair(scales_bar(buffer), static_cast<uint16_t>(1u << leader));
          } else {
            ptx::umma_commit_1cta(scales_bar(buffer));
          }
        }
        __syncwarp();
        desc += T::kStageBytes >> 4;
        if (++stage == args.stages) {
          stage = 0;
          phase ^= 1u;
          desc = desc0;
        }
        if (++buffer == T::kScaleBuffers) buffer = 0;
      }
    }
    __syncwarp();
  } else {
    const int q = warp & 3;
    const uint32_t slab0 = slab_base + static_cast<uint32_t>(q * args.slab_bytes);
    const uint32_t leader_drained = PAIR ? ptx::map_to_cta(drained_bar(0), leader) : drained_bar(0);
    constexpr int kChunk = BN < 32 ? BN : 32;
    constexpr int kChunks = BN / kChunk;
    constexpr int kFirst = T::kOverlap / 32;  // chunks that are handed back early
    int turn = 0;
    uint32_t stores = 0;
    for (int tile = cluster; tile < args.sched.num_tiles; tile += args.sched.num_workers, ++turn) {
      const TileCoord tc = tile_coord(args.sched, tile);
      const int acc = turn & 1;
      const int r_warp = tc.m * T::kTileRows + static_cast<int>(cta) * 128 + q * 32;  // this warp's first row
      const int row = r_warp + static_cast<int>(lane);
      const int s0 = tc.n * BN;
      if (!mx_warp_wait(done_bar(acc), static_cast<uint32_t>(turn >> 1) & 1u)) {
        if (lane == 0) mx_report_timeout(args.status, kStatusEpilogueTimeout, tile, acc, abort_flag);
        break;
      }
      ptx::tc_fence_after_sync();
      const uint32_t taddr = tmem_base + (acc ? T::kAcc1 : 0) + (static_cast<uint32_t>(q * 32) << 16);
      auto hand_back = [&]() {
        ptx::tc_fence_before_sync();
        __syncwarp();
        if (lane == 0) {
          ptx::mbar_arrive_cluster(leader_drained + 8u * static_cast<uint32_t>(T::kOverlap > 0 ? 0 : acc));
        }
      };
      if (args.split > 1) {
        // Partial tile, column by column (the lanes of a warp write consecutive floats), over the ring:
        // every load into it has been consumed. The cluster finishes it below.
#pragma unroll 1
        for (int c = 0; c < BN; c += kChunk) {
          uint32_t v[kChunk];
          ptx::tmem_ld_cols(taddr + c, v);
          ptx::tmem_ld_wait();
#pragma unroll
          for (int j = 0; j < kChunk; ++j) {
            ptx::st_shared_f32(smem_base + static_cast<uint32_t>(((c + j) * 128 + q * 32 + lane) * 4), __uint_as_float(v[j]));
          }
        }
        break;
      }
      const bool live = r_warp < args.R;  // the same for the whole warp
      // The staged rows, columns [c, c + 128) of the tile: whole 16-byte pieces of C by 16 lanes per row, then what
      // lies before and after them, a lane one row.
      auto write_rows = [&](int c) {
        __syncwarp();
        const int cols = min(kMxRowCols, args.S - s0 - c);
        auto at = [&](int r, uint16_t** dst) {
          *dst = args.C + static_cast<long long>(r_warp + r) * args.ldc + s0 + c;
          const int head = static_cast<int>((16u - (reinterpret_cast<uintptr_t>(*dst) & 15u)) & 15u) / 2;
          return head < cols ? head : cols;
        };
#pragma unroll 4
        for (int r = static_cast<int>(lane >> 4); r < 32; r += 2) {
          uint16_t* dst;
          const int e = at(r, &dst) + static_cast<int>(lane & 15u) * 8;
          if (r_warp + r >= args.R || e + 8 > cols) continue;
          const uint32_t src = slab0 + static_cast<uint32_t>(r * kMxRowPitch + (e >> 1) * 4);
          uint32_t w[5];
#pragma unroll
          for (int k = 0; k < 5; ++k) w[k] = (k < 4 || (e & 1)) ? ptx::ld_shared_u32(src + k * 4) : 0u;
          if (e & 1) {
#pragma unroll
            for (int k = 0; k < 4; ++k) w[k] = __funnelshift_r(w[k], w[k + 1], 16);
          }
          *reinterpret_cast<uint4*>(dst + e) = make_uint4(w[0], w[1], w[2], w[3]);
        }
        if (row < args.R) {
          uint16_t* dst;
          const int head = at(static_cast<int>(lane), &dst);
          const int tail = head + (cols - head) / 8 * 8;
          const uint32_t src = slab0 + lane * kMxRowPitch;
          for (int k = 0; k < head; ++k) dst[k] = ptx::ld_shared_u16(src + static_cast<uint32_t>(k * 2));
          for (int k = tail; k < cols; ++k) dst[k] = ptx::ld_shared_u16(src + static_cast<uint32_t>(k * 2));
        }
        __syncwarp();  // before the rows are overwritten
      };
      // One 32-column piece of this lane's row, already in the output type, to C.
      auto store = [&](const uint32_t (&p)[kChunk / 2], int c) {
        if (!live || s0 + c >= args.S) return;
        if (!T::kRowMajor || args.transposed) {
          if (row < args.R) {
#pragma unroll
            for (int j = 0; j < kChunk; ++j) {
              if (s0 + c + j < args.S) {
                args.C[static_cast<long long>(s0 + c + j) * args.ldc + row] = static_cast<uint16_t>(p[j / 2] >> (16 * (j & 1)));
              }
            }
          }
          return;
        }
        if constexpr (T::kRowMajor) {
          if (args.tma_store) {
            // 32 rows x 32 columns as a 64-byte-swizzled box for a TMA store
            const uint32_t slab = slab0 + (stores & (kMxSlabs - 1)) * kMxSlabBytes;
            ++stores;
            if (lane == 0) ptx::tma_store_wait_read<kMxSlabs - 1>();
            __syncwarp();
#pragma unroll
            for (int j = 0; j < kChunk / 8; ++j) {
              ptx::st_shared_v4(slab + lane * 64u + ((static_cast<uint32_t>(j) ^ ((lane >> 1) & 3u)) << 4), p[4 * j], p[4 * j + 1],
                                p[4 * j + 2], p[4 * j + 3]);
            }
            ptx::fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) {
              ptx::tma_store_3d(&map_c, slab, s0 + c, r_warp, 0);
              ptx::tma_store_commit();
            }
          } else {
#pragma unroll
            for (int j = 0; j < kChunk / 8; ++j) {
              ptx::st_shared_v4(slab0 + lane * kMxRowPitch + static_cast<uint32_t>(c % kMxRowCols * 2 + j * 16), p[4 * j],
                                p[4 * j + 1], p[4 * j + 2], p[4 * j + 3]);
            }
            if ((c + kChunk) % kMxRowCols == 0 || s0 + c + kChunk >= args.S) write_rows(c / kMxRowCols * kMxRowCols);
          }
        }
      };
      auto pack = [&](const uint32_t (&v)[kChunk], uint32_t (&p)[kChunk / 2]) {
#pragma unroll
        for (int j = 0; j < kChunk / 2; ++j) {
          p[j] = mx_pack16<F16>(mx_finish(args, __uint_as_float(v[2 * j])), mx_finish(args, __uint_as_float(v[2 * j + 1])));
        }
      };
      auto store_rest = [&](int c_begin, int c_end) {
#pragma unroll 1
        for (int c = c_begin; c < c_end; c += kChunk) {
          uint32_t v[kChunk], p[kChunk / 2];
          __syncwarp();
          ptx::tmem_ld_cols(taddr + c, v);
          ptx::tmem_ld_wait();
          if (kFirst == 0 && c + kChunk == BN) hand_back();
          pack(v, p);
          store(p, c);
        }
      };
      if constexpr (kFirst > 0) {
        // The overlapping chunks, the last ones of the first accumulator or the first of the second, are read out
        // and handed back before anything is stored: the next tile waits for no more than this. Stores go from left to right.
        const int c_first = acc ? 0 : BN - T::kOverlap;
        uint32_t p[kFirst][kChunk / 2];
#pragma unroll
        for (int i = 0; i < kFirst; ++i) {
          uint32_t v[kChunk];
          ptx::tmem_ld_cols(taddr + c_first + i * kChunk, v);
          ptx::tmem_ld_wait();
          pack(v, p[i]);
        }
        hand_back();
        if (acc == 0) store_rest(0, c_first);
#pragma unroll
        for (int i = 0; i < kFirst; ++i) store(p[i], c_first + i * kChunk);
        if (acc == 1) store_rest(T::kOverlap, BN);
      } else {
        store_rest(0, BN);
      }
    }
    if (T::kRowMajor && lane == 0) ptx::tma_store_wait<0>();
    __syncwarp();
  }

  if (args.split > 1) {
    __syncwarp();
    ptx::cluster_arrive();
    ptx::cluster_wait();
    if (*abort_flag == 0u) {
      // Part p finishes columns [BN * p / split, BN * (p + 1) / split): a warp one column at a time, a lane
      // four rows of it, four columns on the way (one at a time is a remote latency per column: 25 us for 128).
      const TileCoord tc = tile_coord(args.sched, cluster);
      const int s0 = tc.n * BN;
      const int row = tc.m * T::kTileRows + static_cast<int>(cta) * 128 + static_cast<int>(lane) * 4;
      const int c0 = BN * part / args.split;
      const int c1 = min(BN * (part + 1) / args.split, args.S - s0);
      const bool wide = row + 4 <= args.R && args.ldc % 4 == 0 && (reinterpret_cast<uintptr_t>(args.C) & 7u) == 0;
      constexpr int kWarps = T::kThreads / 32, kAhead = 4;
      for (int c = c0 + warp; c < c1 && row < args.R; c += kWarps * kAhead) {
        float4 sum[kAhead];
#pragma unroll
        for (int u = 0; u < kAhead; ++u) sum[u] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        for (int p = 0; p < args.split; ++p) {
          const uint32_t peer = ptx::map_to_cta(smem_base, p * G + cta);
#pragma unroll
          for (int u = 0; u < kAhead; ++u) {
            if (c + u * kWarps < c1) {
              const float4 v = ptx::ld_cluster_v4(peer + static_cast<uint32_t>(((c + u * kWarps) * 128 + lane * 4) * 4));
              sum[u].x += v.x;
              sum[u].y += v.y;
              sum[u].z += v.z;
              sum[u].w += v.w;
            }
          }
        }
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
          if (c + u * kWarps >= c1) break;
          uint16_t* dst = args.C + static_cast<long long>(s0 + c + u * kWarps) * args.ldc + row;
          const uint32_t lo = mx_pack16<F16>(mx_finish(args, sum[u].x), mx_finish(args, sum[u].y));
          const uint32_t hi = mx_pack16<F16>(mx_finish(args, sum[u].z), mx_finish(args, sum[u].w));
          if (wide) {
            *reinterpret_cast<uint2*>(dst) = make_uint2(lo, hi);
          } else {
#pragma unroll
            for (int h = 0; h < 4; ++h) {
              if (row + h < args.R) dst[h] = static_cast<uint16_t>((h < 2 ? lo : hi) >> (16 * (h & 1)));
            }
          }
        }
      }
    }
    __syncwarp();
  }

  ptx::tc_fence_before_sync();
  __syncthreads();
  if (*abort_flag != 0u) {
    // A wait gave up: let copies in flight land before shared and tensor memory are released.
    for (int i = 0; i < 1000; ++i) __nanosleep(1000);
  }
  if (cluster_size > 1) {
    // No CTA leaves while another reads its partial tile, its barriers or its tensor memory.
    ptx::cluster_arrive();
    ptx::cluster_wait();
  }
  if (warp == 1) {
    ptx::tc_fence_after_sync();
    ptx::tmem_dealloc<G>(tmem_base, T::kTmemCols);
  }
}

}  // namespace b200
