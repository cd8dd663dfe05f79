// Host side of the microscaled 4-bit operators (include/b200_gemm.h): quantisation, its inverse, and the product.
#include <cstring>

#include "internal.h"
#include "sm100/mx_gemm.cuh"
#include "sm100/mx_quant.cuh"

namespace {

using namespace b200;

bool format_known(int format) { return format == B200_MXFP4 || format == B200_NVFP4; }

// Powers of two within fp32's comfortable range, so that dividing by one is exact.
bool tensor_scale_ok(int format, float t) {
  uint32_t bits;
  std::memcpy(&bits, &t, sizeof bits);
  const int exponent = static_cast<int>(bits >> 23) - 127;
  if ((bits & 0x807FFFFFu) != 0 || exponent < -64 || exponent > 64) return false;
  return format == B200_NVFP4 || t == 1.0f;
}

template <int FMT, int F16, int ROW, int COL>
int launch_quantize(const QuantArgs& args, bool vec, long long grid, cudaStream_t stream) {
  Launch l(grid, kQuantThreads, 0, stream);
  if (vec) {
    B200_TRY_CUDA(cudaLaunchKernelEx(&l.config, &quantize_kernel<FMT, F16, ROW, COL, 1>, args));
  } else {
    B200_TRY_CUDA(cudaLaunchKernelEx(&l.config, &quantize_kernel<FMT, F16, ROW, COL, 0>, args));
  }
  return B200_OK;
}

template <int FMT, int F16>
int launch_quantize(const QuantArgs& args, bool vec, long long grid, cudaStream_t stream) {
  if (args.data[0] && args.data[1]) return launch_quantize<FMT, F16, 1, 1>(args, vec, grid, stream);
  if (args.data[0]) return launch_quantize<FMT, F16, 1, 0>(args, vec, grid, stream);
  return launch_quantize<FMT, F16, 0, 1>(args, vec, grid, stream);
}

template <int FMT, int F16>
int launch_dequantize(const DequantArgs& args, bool vec, long long grid, cudaStream_t stream) {
  Launch l(grid, kQuantThreads, 0, stream);
  if (vec) {
    B200_TRY_CUDA(cudaLaunchKernelEx(&l.config, &dequantize_kernel<FMT, F16, 1>, args));
  } else {
    B200_TRY_CUDA(cudaLaunchKernelEx(&l.config, &dequantize_kernel<FMT, F16, 0>, args));
  }
  return B200_OK;
}

// Rank-3 tile map {inner, rows, 1}.
int tile_map(const DeviceInfo& dev, CUtensorMap* out, CUtensorMapDataType type, const void* base, uint64_t inner,
             uint64_t rows, uint64_t pitch_bytes, uint32_t box_inner, uint32_t box_rows, CUtensorMapSwizzle swizzle) {
  cuuint64_t dims[3] = {inner, rows, 1};
  cuuint64_t strides[2] = {pitch_bytes, pitch_bytes * rows};
  cuuint32_t box[3] = {box_inner, box_rows, 1};
  cuuint32_t steps[3] = {1, 1, 1};
  const CUresult r = dev.encode(out, type, 3, const_cast<void*>(base), dims, strides, box, steps,
                                CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                                CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? B200_OK : cuda_failed(static_cast<int>(r));
}

int code_map(const DeviceInfo& dev, CUtensorMap* out, const void* codes, long long rows, long long cols, int box_rows) {
  const uint64_t pitch = static_cast<uint64_t>(mx_pitch(cols));
  return tile_map(dev, out, CU_TENSOR_MAP_DATA_TYPE_UINT8, codes, pitch, static_cast<uint64_t>(rows), pitch, 128,
                  static_cast<uint32_t>(box_rows), CU_TENSOR_MAP_SWIZZLE_128B);
}

// The scales as rows of 1 KB; one box is one 128 x 256 tile's scales.
int scale_map(const DeviceInfo& dev, CUtensorMap* out, int format, const void* scales, long long rows, long long cols) {
  const uint64_t kilobytes = static_cast<uint64_t>(mx_scale_bytes(format, rows, cols) / 1024);
  return tile_map(dev, out, CU_TENSOR_MAP_DATA_TYPE_UINT32, scales, 256, kilobytes, 1024, 256,
                  static_cast<uint32_t>(mx_tile_bytes(format) / 1024), CU_TENSOR_MAP_SWIZZLE_NONE);
}

struct MxProduct {
  int R, S, K;
  const void *x, *sx, *w, *sw;
};

// How a product is cut: CTAs of 128 x BN or pairs of 256 x BN, and the K ranges that share a tile.
struct MxPlan {
  int width;       // BN
  int pair;
  int transposed;
  int split;
};

long long ceil_div(long long a, long long b) { return (a + b - 1) / b; }

// The cut by shape. Up to 64 rows of A ride on the MMA's N in the narrowest tile that holds them, and 128 weight
// rows per CTA: two CTAs per SM, so that up to 296 tiles stream at a time. Beyond, CTA pairs: 256 weight
// rows against 128 or 256 rows of A while that leaves pairs idle (then K is shared out), else 256
// rows of A against 256 weight rows, row-major.
MxPlan plan_product(int M, int N, int K, int sms) {
  const long long k_tiles = mx_col_tiles(K);
  MxPlan p{};
  p.transposed = 1;
  p.split = 1;
  if (M <= 64) {
    p.width = M <= 16 ? 16 : M <= 32 ? 32 : 64;
    const long long tiles = ceil_div(N, 128);
    while (p.split < 8 && tiles * (p.split + 1) <= 2ll * sms && k_tiles >= 4ll * (p.split + 1)) ++p.split;
    return p;
  }
  p.pair = 1;
  p.width = M <= 128 ? 128 : 256;
  const long long tiles = ceil_div(N, 256) * ceil_div(M, p.width);
  while (p.split < 4 && tiles * (p.split + 1) <= sms / 2 && k_tiles >= 4ll * (p.split + 1)) ++p.split;
  if (p.split == 1 && M > 256) {
    p.transposed = 0;
    // Lone CTAs of 128 x 256 take about 1.2 times as long for their share (they load all of B's tile themselves:
    // 4096 x 8192 x 4096 NVFP4 69 against 58 us), but halve what a partly filled last wave wastes
    // (777 x 5008 x 4104: 80 tiles are two waves of 74 pairs, 140 half tiles one wave of 148, 16.1 against 21.3 us).
    const long long pair_waves = ceil_div(tiles, sms / 2);
    const long long lone_waves = ceil_div(ceil_div(M, 128) * ceil_div(N, 256), sms);
    if (lone_waves * 6 < pair_waves * 5) p.pair = 0;
  }
  return p;
}

template <int FMT, int BN, int PAIR, int F16>
int launch_gemm(const DeviceInfo& dev, const MxProduct& p, const MxPlan& plan, MxGemmArgs args, cudaStream_t stream) {
  using T = MxGemmTraits<FMT, BN, PAIR>;
  if (!T::kRowMajor && !plan.transposed) return B200_ERR_INVALID_ARG;  // (plan_product never asks for it)
  args.k_tiles = static_cast<int>(mx_col_tiles(p.K));
  args.split = plan.split;
  args.tma_store = !plan.transposed && aligned16(args.C) && args.ldc % 8 == 0 ? 1 : 0;
  args.slab_bytes = plan.transposed ? 0 : args.tma_store ? kMxSlabs * kMxSlabBytes : 32 * kMxRowPitch;
  args.sched.tiles_m = static_cast<int>(ceil_div(p.R, T::kTileRows));
  args.sched.tiles_n = static_cast<int>(ceil_div(p.S, BN));
  args.sched.batch = 1;
  const long long tiles = static_cast<long long>(args.sched.tiles_m) * args.sched.tiles_n;
  if (tiles > 0x7FFFFFFFll / 16) return B200_ERR_INVALID_ARG;
  args.sched.num_tiles = static_cast<int>(tiles);
  args.sched.k_tiles = args.k_tiles;
  args.sched.group = 8;
  args.sched.mode = kDataParallel;
  args.sched.split_k = 1;
  // Two lone CTAs to an SM where their rings and accumulators fit: 113 KB of shared memory and half of tensor
  // memory each.
  const bool two = !PAIR && T::kTmemCols <= 256;
  const long long workers = static_cast<long long>(dev.sm_count) * (two ? 2 : 1) / T::kCtas;
  const long long waves = ceil_div(tiles, workers);
  args.sched.num_workers = static_cast<int>(plan.split > 1 ? tiles : ceil_div(tiles, waves));
  const int budget = two ? 113 * 1024 : dev.smem_optin;
  int stages = (budget - T::smem_bytes(0, args.slab_bytes)) / T::kStageBytes;
  if (stages > kMxMaxStages) stages = kMxMaxStages;
  if (stages < T::kScaleBuffers || (plan.split > 1 && stages * T::kStageBytes < BN * 512)) return B200_ERR_SMEM;
  args.stages = stages;
  CUtensorMap mx, mw, msx, msw, mc;
  int rc = code_map(dev, &mx, p.x, p.R, p.K, 128);
  if (rc == B200_OK) rc = code_map(dev, &mw, p.w, p.S, p.K, T::kWRows);
  if (rc == B200_OK) rc = scale_map(dev, &msx, FMT, p.sx, p.R, p.K);
  if (rc == B200_OK) rc = scale_map(dev, &msw, FMT, p.sw, p.S, p.K);
  if (rc != B200_OK) return rc;
  if (args.tma_store) {
    rc = tile_map(dev, &mc, CU_TENSOR_MAP_DATA_TYPE_UINT16, args.C, static_cast<uint64_t>(p.S), static_cast<uint64_t>(p.R),
                  static_cast<uint64_t>(args.ldc) * 2, 32, 32, CU_TENSOR_MAP_SWIZZLE_64B);
    if (rc != B200_OK) return rc;
  } else {
    mc = mx;  // never followed
  }
  const auto kernel = &mx_gemm_kernel<FMT, BN, PAIR, F16>;
  static std::atomic<bool> allowed[64];
  rc = allow_shared_memory(dev, kernel, allowed);
  if (rc != B200_OK) return rc;
  const int cluster = plan.split * T::kCtas;
  Launch l(static_cast<long long>(args.sched.num_workers) * cluster, T::kThreads,
           static_cast<size_t>(T::smem_bytes(stages, args.slab_bytes)), stream, cluster);
  B200_TRY_CUDA(cudaLaunchKernelEx(&l.config, kernel, mx, mw, msx, msw, mc, args));
  return B200_OK;
}

template <int FMT, int F16>
int launch_gemm(const DeviceInfo& dev, const MxProduct& p, const MxPlan& plan, const MxGemmArgs& args, cudaStream_t stream) {
  switch (plan.width) {
    case 16: return launch_gemm<FMT, 16, 0, F16>(dev, p, plan, args, stream);
    case 32: return launch_gemm<FMT, 32, 0, F16>(dev, p, plan, args, stream);
    case 64: return launch_gemm<FMT, 64, 0, F16>(dev, p, plan, args, stream);
    case 128: return launch_gemm<FMT, 128, 1, F16>(dev, p, plan, args, stream);
    default:
      return plan.pair ? launch_gemm<FMT, 256, 1, F16>(dev, p, plan, args, stream)
                       : launch_gemm<FMT, 256, 0, F16>(dev, p, plan, args, stream);
  }
}

}  // namespace

extern "C" {

size_t b200_mx_data_bytes(int rows, int cols) {
  return rows > 0 && cols > 0 ? static_cast<size_t>(rows * mx_pitch(cols)) : 0;
}

size_t b200_mx_scale_bytes(int format, int rows, int cols) {
  return format_known(format) && rows > 0 && cols > 0 ? static_cast<size_t>(mx_scale_bytes(format, rows, cols)) : 0;
}

int b200_mx_quantize(int format, int f16, int rows, int cols, const void* X, long long ldx, float tensor_scale,
                     void* data, void* scales, void* data_t, void* scales_t, void* stream) {
  if (!format_known(format) || rows <= 0 || cols <= 0 || X == nullptr || ldx < cols) return B200_ERR_INVALID_ARG;
  if ((data == nullptr) != (scales == nullptr) || (data_t == nullptr) != (scales_t == nullptr)) return B200_ERR_INVALID_ARG;
  if (data == nullptr && data_t == nullptr) return B200_ERR_INVALID_ARG;
  if (!aligned16(data) || !aligned16(scales) || !aligned16(data_t) || !aligned16(scales_t)) return B200_ERR_INVALID_ARG;
  if ((reinterpret_cast<uintptr_t>(X) & 1u) || !tensor_scale_ok(format, tensor_scale)) return B200_ERR_INVALID_ARG;
  QuantArgs args;
  args.x = static_cast<const uint16_t*>(X);
  args.rows = rows;
  args.cols = cols;
  args.ldx = ldx;
  args.inv_t = 1.0f / tensor_scale;
  args.data[0] = static_cast<uint8_t*>(data);
  args.data[1] = static_cast<uint8_t*>(data_t);
  args.scales[0] = static_cast<uint8_t*>(scales);
  args.scales[1] = static_cast<uint8_t*>(scales_t);
  args.pitch[0] = mx_pitch(cols);
  args.pitch[1] = mx_pitch(rows);
  args.col_tiles[0] = mx_col_tiles(cols);
  args.col_tiles[1] = mx_col_tiles(rows);
  args.row_tiles[0] = mx_row_tiles(rows);
  args.row_tiles[1] = mx_row_tiles(cols);
  const long long tiles_x = data != nullptr ? 2 * args.col_tiles[0] : args.row_tiles[1];
  const long long tiles_y = data_t != nullptr ? 2 * args.col_tiles[1] : args.row_tiles[0];
  if (tiles_x * tiles_y > 0x7FFFFFFFll) return B200_ERR_INVALID_ARG;
  args.tiles_x = static_cast<int>(tiles_x);
  DeviceInfo dev;
  const int rc = device_info(&dev);
  if (rc != B200_OK) return rc;
  const bool vec = aligned16(X) && ldx % 8 == 0;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const long long grid = tiles_x * tiles_y;
  if (format == B200_MXFP4) {
    return f16 ? launch_quantize<kMxfp4, 1>(args, vec, grid, s) : launch_quantize<kMxfp4, 0>(args, vec, grid, s);
  }
  return f16 ? launch_quantize<kNvfp4, 1>(args, vec, grid, s) : launch_quantize<kNvfp4, 0>(args, vec, grid, s);
}

int b200_mx_dequantize(int format, int f16, int rows, int cols, const void* data, const void* scales, float tensor_scale,
                       void* X, long long ldx, void* stream) {
  if (!format_known(format) || rows <= 0 || cols <= 0 || X == nullptr || ldx < cols) return B200_ERR_INVALID_ARG;
  if (data == nullptr || scales == nullptr || !aligned16(data) || !aligned16(scales)) return B200_ERR_INVALID_ARG;
  if ((reinterpret_cast<uintptr_t>(X) & 1u) != 0) return B200_ERR_INVALID_ARG;
  if (!(tensor_scale > 0.0f) || tensor_scale > 3.4e38f || (format == B200_MXFP4 && tensor_scale != 1.0f)) return B200_ERR_INVALID_ARG;
  DequantArgs args;
  args.data = static_cast<const uint8_t*>(data);
  args.scales = static_cast<const uint8_t*>(scales);
  args.rows = rows;
  args.cols = cols;
  args.pitch = mx_pitch(cols);
  args.col_tiles = mx_col_tiles(cols);
  args.tensor_scale = tensor_scale;
  uint32_t bits;
  std::memcpy(&bits, &tensor_scale, sizeof bits);
  args.inexact = (bits & 0x007FFFFFu) != 0 ? 1 : 0;
  args.x = static_cast<uint16_t*>(X);
  args.ldx = ldx;
  const long long tiles_x = (cols + kQuantTile - 1) / kQuantTile, tiles_y = mx_row_tiles(rows);
  if (tiles_x * tiles_y > 0x7FFFFFFFll) return B200_ERR_INVALID_ARG;
  args.tiles_x = static_cast<int>(tiles_x);
  DeviceInfo dev;
  const int rc = device_info(&dev);
  if (rc != B200_OK) return rc;
  const bool vec = aligned16(X) && ldx % 8 == 0;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const long long grid = tiles_x * tiles_y;
  if (format == B200_MXFP4) {
    return f16 ? launch_dequantize<kMxfp4, 1>(args, vec, grid, s) : launch_dequantize<kMxfp4, 0>(args, vec, grid, s);
  }
  return f16 ? launch_dequantize<kNvfp4, 1>(args, vec, grid, s) : launch_dequantize<kNvfp4, 0>(args, vec, grid, s);
}

int b200_gemm_mx(int format, int f16, int M, int N, int K, const void* A, const void* A_scales, const void* B,
                 const void* B_scales, void* C, float alpha, float beta, void* stream) {
  if (!format_known(format) || M <= 0 || N <= 0 || K <= 0) return B200_ERR_INVALID_ARG;
  if (M > 0x7FFFFFFF - 512 || N > 0x7FFFFFFF - 512 || K > 0x7FFFFFFF - 512) return B200_ERR_INVALID_ARG;  // (tiles end in 32 bits)
  if (A == nullptr || A_scales == nullptr || B == nullptr || B_scales == nullptr || C == nullptr) return B200_ERR_INVALID_ARG;
  if (!aligned16(A) || !aligned16(A_scales) || !aligned16(B) || !aligned16(B_scales)) return B200_ERR_INVALID_ARG;
  if ((reinterpret_cast<uintptr_t>(C) & 1u) != 0) return B200_ERR_INVALID_ARG;
  if (mx_scale_bytes(format, M, K) / 1024 > 0x7FFFFFFFll || mx_scale_bytes(format, N, K) / 1024 > 0x7FFFFFFFll) {
    return B200_ERR_INVALID_ARG;
  }
  DeviceInfo dev;
  const int rc = device_info(&dev);
  if (rc != B200_OK) return rc;
  const MxPlan plan = plan_product(M, N, K, dev.sm_count);
  MxProduct p;
  MxGemmArgs args;
  std::memset(&args, 0, sizeof args);
  if (plan.transposed) {
    p = MxProduct{N, M, K, B, B_scales, A, A_scales};
  } else {
    p = MxProduct{M, N, K, A, A_scales, B, B_scales};
  }
  args.R = p.R;
  args.S = p.S;
  args.transposed = plan.transposed;
  args.C = static_cast<uint16_t*>(C);
  args.ldc = N;
  args.alpha = alpha;
  args.beta = beta;
  args.scale = (alpha != 1.0f || beta != 0.0f) ? 1 : 0;
  args.status = dev.status;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (format == B200_MXFP4) {
    return f16 ? launch_gemm<kMxfp4, 1>(dev, p, plan, args, s) : launch_gemm<kMxfp4, 0>(dev, p, plan, args, s);
  }
  return f16 ? launch_gemm<kNvfp4, 1>(dev, p, plan, args, s) : launch_gemm<kNvfp4, 0>(dev, p, plan, args, s);
}

}  // extern "C"
