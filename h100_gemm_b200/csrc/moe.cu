// Host side of the mixture-of-experts layer (include/b200_gemm.h).
#include <cstring>

#include "internal.h"
#include "sm100/moe.cuh"

namespace {

using namespace b200;

size_t round_up(size_t x) { return (x + 255) / 256 * 256; }

// Workspace: [h][ids][weights]
size_t h_bytes(int T, int k, int I) { return round_up(static_cast<size_t>(T) * k * I * 4); }
size_t pair_bytes(int T, int k) { return round_up(static_cast<size_t>(T) * k * 4); }

bool sizes_ok(int T, int E, int k, int H, int I) {
  return T >= 1 && T <= kMoeMaxTokens && E >= 1 && E <= kMoeMaxExperts && k >= 1 && k <= kMoeMaxTopK && k <= E && H >= 8 &&
         I >= 8 && H % 8 == 0 && I % 8 == 0 && H <= (1 << 20) && I <= (1 << 20);
}

// What b200_mx_dequantize takes.
bool weights_scale_ok(int format, float t) { return t > 0.0f && t <= 3.4e38f && (format == B200_NVFP4 || t == 1.0f); }

// lift (a power of two) times the tensor scale in one number, unless that leaves fp32's range: then 2^32 of it apart.
void split_factor(float (&factor)[2], float lift, float tensor_scale) {
  factor[0] = lift * tensor_scale;
  factor[1] = 1.0f;
  if (factor[0] > 3.4e38f) {
    factor[0] = tensor_scale * (lift * 0x1p-32f);
    factor[1] = 0x1p32f;
  }
}

template <int W, int F16>
int launch_all(const DeviceInfo& dev, const MoeArgs& args, cudaStream_t stream) {
  static std::atomic<bool> up_allowed[64], down_allowed[64];
  int rc = allow_shared_memory(dev, &moe_gate_up_kernel<W, F16>, up_allowed);
  if (rc == B200_OK) rc = allow_shared_memory(dev, &moe_down_kernel<W, F16>, down_allowed);
  if (rc != B200_OK) return rc;

  // As few tokens to a cluster as 8 clusters allow, which an idle device takes at once (4 tokens one to a cluster: the layer
  // 1.9 us shorter than with all four in one); then up to kRouterTokens, so that the router's rows are not read too often.
  const int group = args.T <= 8 ? 1 : args.T <= 16 ? 2 : kRouterTokens;
  const int clusters = (args.T + group - 1) / group;
  // 16 warps fill an SM with their registers: beyond 8 clusters two smaller CTAs per SM keep all of them resident
  // (64 tokens, 128 experts: 8.4 against 10.5 us; 4 tokens in one cluster: 6.8 against 6.1 us).
  const int threads = clusters > 8 ? kRouterThreads / 2 : kRouterThreads;
  Launch route(clusters * kRouterCluster, threads, 0, stream, kRouterCluster);
  if (group == 1) {
    B200_TRY_CUDA(cudaLaunchKernelEx(&route.config, &moe_router_kernel<F16, 1>, args));
  } else if (group == 2) {
    B200_TRY_CUDA(cudaLaunchKernelEx(&route.config, &moe_router_kernel<F16, 2>, args));
  } else {
    B200_TRY_CUDA(cudaLaunchKernelEx(&route.config, &moe_router_kernel<F16, kRouterTokens>, args));
  }

  constexpr int MT = MoeUnit<W, F16>::kTiles;
  using Hidden = Down<W, F16>;
  const int tables = route_table_bytes(args.E, args.T * args.k);
  const int most = args.T * args.k < args.E ? args.T * args.k : args.E;  // experts that can be chosen
  const long long units = static_cast<long long>(most) * ((args.I + 8 * MT - 1) / (8 * MT));
  Launch up(static_cast<int>(units < 2ll * dev.sm_count ? units : 2ll * dev.sm_count), kMoeThreads,
            gate_up_buffers(MT, args.T) * kMoeWarps * gate_up_stride(MT, args.T) * 16 + tables, stream, 1);
  B200_TRY_CUDA(cudaLaunchKernelEx(&up.config, &moe_gate_up_kernel<W, F16>, args));

  // Clusters share the columns of a unit until every SM has two CTAs, but no warp is left without a step.
  const int columns = (args.H + 16 * Hidden::MT - 1) / (16 * Hidden::MT);
  const long long steps = static_cast<long long>(most) * ((args.I + Hidden::kStep - 1) / Hidden::kStep);
  int split = 1;
  while (split < 8 && columns * split * 2 <= dev.sm_count * 2 && steps >= 2ll * split * kMoeWarps) split *= 2;
  Launch down(columns * split, kMoeThreads, (kMoeWarps * args.T * Hidden::kPitch * 4 + 15) / 16 * 16 + tables, stream,
              split);
  B200_TRY_CUDA(cudaLaunchKernelEx(&down.config, &moe_down_kernel<W, F16>, args, split));
  return B200_OK;
}

}  // namespace

extern "C" {

size_t b200_moe_workspace_bytes(int T, int E, int top_k, int H, int I) {
  return sizes_ok(T, E, top_k, H, I) ? h_bytes(T, top_k, I) + 2 * pair_bytes(T, top_k) : 0;
}

int b200_moe_layer(int f16, int T, int E, int top_k, int H, int I, const void* X, const void* router, const float* bias,
                   int weight_format, const void* W1, const void* W1_scales, float W1_tensor_scale, const void* W2,
                   const void* W2_scales, float W2_tensor_scale, int renormalize, void* out, int* ids, float* weights,
                   void* workspace, size_t workspace_bytes, void* stream) {
  if (!sizes_ok(T, E, top_k, H, I)) return B200_ERR_INVALID_ARG;
  const bool four_bit = weight_format != B200_MOE_16BIT;
  if (weight_format != B200_MOE_16BIT && weight_format != B200_MXFP4 && weight_format != B200_NVFP4) return B200_ERR_INVALID_ARG;
  if (four_bit && f16) return B200_ERR_INVALID_ARG;
  if (X == nullptr || router == nullptr || W1 == nullptr || W2 == nullptr || out == nullptr) return B200_ERR_INVALID_ARG;
  if (four_bit && (W1_scales == nullptr || W2_scales == nullptr)) return B200_ERR_INVALID_ARG;
  if (four_bit && !(weights_scale_ok(weight_format, W1_tensor_scale) && weights_scale_ok(weight_format, W2_tensor_scale))) {
    return B200_ERR_INVALID_ARG;
  }
  if (!aligned16(X) || !aligned16(router) || !aligned16(W1) || !aligned16(W2) || !aligned16(W1_scales) ||
      !aligned16(W2_scales) || (reinterpret_cast<uintptr_t>(out) & 1u) || (reinterpret_cast<uintptr_t>(bias) & 3u) ||
      (reinterpret_cast<uintptr_t>(ids) & 3u) || (reinterpret_cast<uintptr_t>(weights) & 3u)) {
    return B200_ERR_INVALID_ARG;
  }
  if (workspace == nullptr || workspace_bytes < b200_moe_workspace_bytes(T, E, top_k, H, I)) return B200_ERR_WORKSPACE;
  if (reinterpret_cast<uintptr_t>(workspace) & 255u) return B200_ERR_INVALID_ARG;
  DeviceInfo dev;
  const int rc = device_info(&dev);
  if (rc != B200_OK) return rc;
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  MoeArgs args;
  std::memset(&args, 0, sizeof args);
  args.T = T;
  args.E = E;
  args.k = top_k;
  args.H = H;
  args.I = I;
  args.renormalize = renormalize ? 1 : 0;
  args.x = static_cast<const uint16_t*>(X);
  args.router = static_cast<const uint16_t*>(router);
  args.bias = bias;
  args.w1.data = static_cast<const uint8_t*>(W1);
  args.w1.scales = static_cast<const uint8_t*>(W1_scales);
  args.w1.pitch = four_bit ? mx_pitch(H) : 2ll * H;
  args.w1.col_tiles = mx_col_tiles(H);
  args.w2.data = static_cast<const uint8_t*>(W2);
  args.w2.scales = static_cast<const uint8_t*>(W2_scales);
  args.w2.pitch = four_bit ? mx_pitch(I) : 2ll * I;
  args.w2.col_tiles = mx_col_tiles(I);
  const float lift = weight_format == B200_NVFP4 ? MoeUnit<kMoeNvfp4, 0>::kLift : 1.0f;
  split_factor(args.scale1, lift, four_bit ? W1_tensor_scale : 1.0f);
  split_factor(args.scale2, lift, four_bit ? W2_tensor_scale : 1.0f);
  args.h = reinterpret_cast<uint16_t*>(ws);
  args.ids = ids != nullptr ? ids : reinterpret_cast<int*>(ws + h_bytes(T, top_k, I));
  args.weights = weights != nullptr ? weights : reinterpret_cast<float*>(ws + h_bytes(T, top_k, I) + pair_bytes(T, top_k));
  args.out = static_cast<uint16_t*>(out);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (weight_format == B200_MXFP4) return launch_all<kMoeMxfp4, 0>(dev, args, s);
  if (weight_format == B200_NVFP4) return launch_all<kMoeNvfp4, 0>(dev, args, s);
  return f16 ? launch_all<kMoe16, 1>(dev, args, s) : launch_all<kMoe16, 0>(dev, args, s);
}

}  // extern "C"
