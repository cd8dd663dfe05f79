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
//   warp 1      MMA issuer: scales to tensor memory, four MMAs of K = 64 per K-tile
//   warps 2-5   epilogue: accumulator -> registers -> C
//
// One CTA computes a 128 x BN tile, X's rows on the MMA's M. With few rows in the caller's A the operands are
// swapped (C is written transposed): weights on M, the rows on N, so that no tensor work and no
// accumulator is spent on padding. When there are fewer tiles than SMs a cluster of CTAs shares one
// tile, each taking a range of K; the partial tiles are added over distributed shared memory in rank order, so that
// no workspace is needed, nothing depends on timing and a captured launch can be replayed.
#pragma once

#include "desc.cuh"
#include "mx_format.cuh"
#include "ptx.cuh"
#include "status.cuh"

namespace b200 {

struct MxGemmArgs {
  int R, S;           // rows of X and W
  int k_tiles;        // K-tiles of 256 elements
  int tiles_r;        // tiles along R
  int stages;
  int transposed;     // 1: element (r, s) goes to C[s * ldc + r]
  int vec;            // 1: rows of C start on 16 bytes and S is a multiple of 8
  uint16_t* C;
  long long ldc;
  float alpha, beta;
  int scale;          // 1: C = acc * alpha + beta
  unsigned int* status;
};

static constexpr int kMxMaxStages = 16;
static constexpr int kMxScaleBuffers = 3;  // K-tiles whose scales tensor memory holds at a time (the ring has no fewer stages)

template <int FMT, int BN>
struct MxGemmTraits {
  static constexpr int kThreads = 192;
  static constexpr int kSBlocks = (BN + 127) / 128;                 // scale tiles of W per K-tile
  static constexpr int kXBytes = 128 * 128;
  static constexpr int kWBytes = BN * 128;
  static constexpr int kScaleTile = mx_tile_bytes(FMT);
  static constexpr int kGroups = mx_tile_groups(FMT);
  static constexpr int kStageBytes = kXBytes + kWBytes + (1 + kSBlocks) * kScaleTile;
  static constexpr int kAccCols = BN < 32 ? 32 : BN;
  static constexpr int kScaleCols = kGroups * 4 * (1 + kSBlocks);   // of one K-tile: X's, then W's
  static constexpr int kNeedCols = kAccCols + kMxScaleBuffers * kScaleCols;
  static constexpr int kTmemCols = kNeedCols <= 128 ? 128 : kNeedCols <= 256 ? 256 : 512;
  static_assert(kNeedCols <= 512, "accumulator and scales exceed tensor memory");
  static_assert(BN % 16 == 0 && BN <= 256, "width of the MMA");
  static constexpr int kBarrierBytes = 512;
  static constexpr int smem_bytes(int stages) { return 1024 + stages * kStageBytes + kBarrierBytes; }
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

// Grid: tiles * split CTAs, clusters of `split`; CTA rank r of a cluster takes K-tiles
// [k_tiles * r / split, k_tiles * (r + 1) / split).
template <int FMT, int BN, int F16>
__global__ void __launch_bounds__(192) mx_gemm_kernel(const __grid_constant__ CUtensorMap map_x,
                                                       const __grid_constant__ CUtensorMap map_w,
                                                       const __grid_constant__ CUtensorMap map_sx,
                                                       const __grid_constant__ CUtensorMap map_sw,
                                                       const __grid_constant__ MxGemmArgs args, int split) {
  using T = MxGemmTraits<FMT, BN>;
  extern __shared__ uint8_t smem_raw[];
  const int warp = __shfl_sync(0xffffffffu, static_cast<int>(threadIdx.x) / 32, 0);
  const uint32_t lane = ptx::lane_id();
  const int rank = split > 1 ? static_cast<int>(ptx::cluster_ctarank()) : 0;
  const int tile = static_cast<int>(blockIdx.x) / split;
  const int r0 = (tile % args.tiles_r) * 128;
  const int s0 = (tile / args.tiles_r) * BN;
  const int kt0 = static_cast<int>(static_cast<long long>(args.k_tiles) * rank / split);
  const int kt1 = static_cast<int>(static_cast<long long>(args.k_tiles) * (rank + 1) / split);

  const uint32_t smem_base = (ptx::smem_u32(smem_raw) + 1023u) & ~1023u;
  const uint32_t bar_base = smem_base + static_cast<uint32_t>(args.stages * T::kStageBytes);
  auto stage_addr = [&](int s) { return smem_base + static_cast<uint32_t>(s * T::kStageBytes); };
  auto full_bar = [&](int s) { return bar_base + 8u * static_cast<uint32_t>(s); };
  auto empty_bar = [&](int s) { return bar_base + 8u * static_cast<uint32_t>(kMxMaxStages + s); };
  const uint32_t done_bar = bar_base + 8u * (2 * kMxMaxStages);
  const uint32_t tmem_slot = done_bar + 8u;
  uint8_t* generic_bar = smem_raw + (bar_base - ptx::smem_u32(smem_raw));
  volatile uint32_t* tmem_ptr = reinterpret_cast<volatile uint32_t*>(generic_bar + 8 * (2 * kMxMaxStages + 1));
  volatile uint32_t* abort_flag = tmem_ptr + 1;

  ptx::grid_launch_dependents();
  if (warp == 0 && lane == 0) {
    ptx::prefetch_tensormap(&map_x);
    ptx::prefetch_tensormap(&map_w);
    ptx::prefetch_tensormap(&map_sx);
    ptx::prefetch_tensormap(&map_sw);
    for (int s = 0; s < args.stages; ++s) {
      ptx::mbar_init(full_bar(s), 1);
      ptx::mbar_init(empty_bar(s), 1);
    }
    ptx::mbar_init(done_bar, 1);
    *abort_flag = 0u;
    ptx::fence_mbar_init();
  }
  if (warp == 1) {
    ptx::tmem_alloc<1>(tmem_slot, T::kTmemCols);
    ptx::tmem_relinquish<1>();
  }
  ptx::tc_fence_before_sync();
  __syncthreads();
  ptx::tc_fence_after_sync();
  const uint32_t tmem_base = *tmem_ptr;
  ptx::grid_dependency_wait();

  if (warp == 0) {
    if (lane == 0) {
      int stage = 0;
      uint32_t phase = 0;
      const int sx_tile = (r0 / kMxTileRows) * args.k_tiles, sw_tile = (s0 / kMxTileRows) * args.k_tiles;
      constexpr int kBoxes = T::kScaleTile / 1024;  // 1 KB rows of the scale maps per tile
      for (int kt = kt0; kt < kt1; ++kt) {
        if (!ptx::mbar_wait(empty_bar(stage), phase ^ 1u)) {
          mx_report_timeout(args.status, kStatusProducerTimeout, tile, kt, abort_flag);
          break;
        }
        const uint32_t full = full_bar(stage), x = stage_addr(stage);
        const uint32_t w = x + T::kXBytes, sx = w + T::kWBytes, sw = sx + T::kScaleTile;
        ptx::mbar_arrive_expect_tx(full, T::kStageBytes);
        ptx::tma_load_3d(x, &map_x, full, kt * 128, r0, 0);
        ptx::tma_load_3d(w, &map_w, full, kt * 128, s0, 0);
        ptx::tma_load_3d(sx, &map_sx, full, 0, (sx_tile + kt) * kBoxes, 0);
#pragma unroll
        for (int b = 0; b < T::kSBlocks; ++b) {
          ptx::tma_load_3d(sw + b * T::kScaleTile, &map_sw, full, 0, (sw_tile + b * args.k_tiles + kt) * kBoxes, 0);
        }
        if (++stage == args.stages) {
          stage = 0;
          phase ^= 1u;
        }
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    if (lane == 0) {
      // 16-element blocks: every MMA has a scale column of its own; 32-element blocks: two MMAs share
      // one, the second starting at its upper byte pair.
      constexpr uint32_t idesc0 = make_instr_desc_mxf4(128, BN, FMT == kMxfp4, 0);
      constexpr uint32_t idesc1 = make_instr_desc_mxf4(128, BN, FMT == kMxfp4, FMT == kMxfp4 ? 2 : 0);
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int kt = kt0; kt < kt1; ++kt) {
        const int i = kt - kt0;
        if (i >= kMxScaleBuffers) {
          // The scales of K-tile i - kMxScaleBuffers are overwritten: its MMAs must have completed.
          const int old = i - kMxScaleBuffers;
          if (!ptx::mbar_wait(empty_bar(old % args.stages), static_cast<uint32_t>(old / args.stages) & 1u)) {
            mx_report_timeout(args.status, kStatusMmaTmemTimeout, tile, kt, abort_flag);
            ok = false;
            break;
          }
        }
        if (!ptx::mbar_wait(full_bar(stage), phase)) {
          mx_report_timeout(args.status, kStatusMmaFullTimeout, tile, kt, abort_flag);
          ok = false;
          break;
        }
        ptx::tc_fence_after_sync();
        const uint32_t x = stage_addr(stage), w = x + T::kXBytes, sx = w + T::kWBytes, sw = sx + T::kScaleTile;
        const uint32_t tsx = tmem_base + T::kAccCols + (i % kMxScaleBuffers) * T::kScaleCols;
        const uint32_t tsw = tsx + T::kGroups * 4;
#pragma unroll
        for (int g = 0; g < T::kGroups; ++g) {
          ptx::tmem_copy_scales<1>(tsx + g * 4, make_smem_desc_scales(sx + g * kMxGroupBytes));
#pragma unroll
          for (int b = 0; b < T::kSBlocks; ++b) {
            ptx::tmem_copy_scales<1>(tsw + (g * T::kSBlocks + b) * 4,
                                     make_smem_desc_scales(sw + b * T::kScaleTile + g * kMxGroupBytes));
          }
        }
        const uint64_t dx = make_smem_desc_sw128(x), dw = make_smem_desc_sw128(w);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int g = FMT == kMxfp4 ? k / 2 : k;
          ptx::umma_mxf4<1, FMT == kNvfp4>(tmem_base, dx + k * kDescKStep, dw + k * kDescKStep, (k & 1) ? idesc1 : idesc0,
                                           tsx + g * 4, tsw + g * 4 * T::kSBlocks, (i > 0 || k > 0) ? 1u : 0u);
        }
        ptx::umma_commit_1cta(empty_bar(stage));
        if (++stage == args.stages) {
          stage = 0;
          phase ^= 1u;
        }
      }
      if (ok) ptx::umma_commit_1cta(done_bar);
    }
    __syncwarp();
  }

  const int q = warp & 3;
  const int row = q * 32 + static_cast<int>(lane);  // of the tile
  bool ready = false;
  if (warp >= 2) {
    ready = __all_sync(0xffffffffu, ptx::mbar_wait(done_bar, 0));
    if (!ready && lane == 0) mx_report_timeout(args.status, kStatusEpilogueTimeout, tile, 0, abort_flag);
    ptx::tc_fence_after_sync();
  }
  const uint32_t taddr = tmem_base + (static_cast<uint32_t>(q * 32) << 16);
  constexpr int kChunk = BN < 32 ? BN : 32;
  if (split > 1) {
    // Partial tile, column by column (the lanes of a warp write consecutive floats), over the ring:
    // every load into it has been consumed.
    if (warp >= 2 && ready) {
#pragma unroll 1
      for (int c = 0; c < BN; c += kChunk) {
        uint32_t v[kChunk];
        ptx::tmem_ld_cols(taddr + c, v);
        ptx::tmem_ld_wait();
#pragma unroll
        for (int j = 0; j < kChunk; ++j) {
          ptx::st_shared_f32(smem_base + static_cast<uint32_t>(((c + j) * 128 + row) * 4), __uint_as_float(v[j]));
        }
      }
    }
    __syncwarp();
    ptx::cluster_arrive();
    ptx::cluster_wait();
    if (warp >= 2 && ready && r0 + row < args.R) {
      // Rank r finishes columns [BN * r / split, BN * (r + 1) / split).
      const int c0 = BN * rank / split, c1 = BN * (rank + 1) / split;
      for (int c = c0; c < c1 && s0 + c < args.S; ++c) {
        float sum = 0.0f;
        for (int p = 0; p < split; ++p) {
          sum += ptx::ld_cluster_f32(ptx::map_to_cta(smem_base + static_cast<uint32_t>((c * 128 + row) * 4), p));
        }
        const uint16_t h = static_cast<uint16_t>(mx_pack16<F16>(mx_finish(args, sum), 0.0f));
        if (args.transposed) {
          args.C[static_cast<long long>(s0 + c) * args.ldc + r0 + row] = h;
        } else {
          args.C[static_cast<long long>(r0 + row) * args.ldc + s0 + c] = h;
        }
      }
    }
    __syncwarp();
    ptx::cluster_arrive();  // no CTA leaves while another still reads its partial tile
    ptx::cluster_wait();
  } else if (warp >= 2 && ready) {
#pragma unroll 1
    for (int c = 0; c < BN; c += kChunk) {
      uint32_t v[kChunk];
      __syncwarp();
      ptx::tmem_ld_cols(taddr + c, v);
      ptx::tmem_ld_wait();
      if (r0 + row >= args.R) {
        // a row of padding
      } else if (args.transposed) {
#pragma unroll
        for (int j = 0; j < kChunk; ++j) {
          if (s0 + c + j < args.S) {
            args.C[static_cast<long long>(s0 + c + j) * args.ldc + r0 + row] =
                static_cast<uint16_t>(mx_pack16<F16>(mx_finish(args, __uint_as_float(v[j])), 0.0f));
          }
        }
      } else {
        uint16_t* dst = args.C + static_cast<long long>(r0 + row) * args.ldc + s0 + c;
#pragma unroll
        for (int j = 0; j < kChunk; j += 8) {
          uint32_t p[4];
#pragma unroll
          for (int h = 0; h < 4; ++h) {
            p[h] = mx_pack16<F16>(mx_finish(args, __uint_as_float(v[j + 2 * h])),
                                  mx_finish(args, __uint_as_float(v[j + 2 * h + 1])));
          }
          if (args.vec) {
            if (s0 + c + j < args.S) *reinterpret_cast<uint4*>(dst + j) = make_uint4(p[0], p[1], p[2], p[3]);
          } else {
#pragma unroll
            for (int h = 0; h < 8; ++h) {
              if (s0 + c + j + h < args.S) dst[j + h] = static_cast<uint16_t>(p[h / 2] >> (16 * (h & 1)));
            }
          }
        }
      }
    }
  }

  ptx::tc_fence_before_sync();
  __syncthreads();
  if (*abort_flag != 0u) {
    // A wait gave up: let copies in flight land before shared and tensor memory are released.
    for (int i = 0; i < 1000; ++i) __nanosleep(1000);
  }
  if (warp == 1) {
    ptx::tc_fence_after_sync();
    ptx::tmem_dealloc<1>(tmem_base, T::kTmemCols);
  }
}

}  // namespace b200
