// A mixture-of-experts layer for a few tokens (T <= 64), in three kernels of one launch sequence.
//
//   logits  l[t, e] = x[t] . R[e] + b[e]                                        (fp32)
//   chosen  S[t] = the k largest logits of t (ties: the lower index; -inf is never chosen)
//   weight  p[t, e] = exp(l[t, e]) / sum of exp(l) over S[t], or over all experts
//   gated   h[t, e] = p[t, e] * silu(G_e x[t]) * (U_e x[t])                     (fp32, rounded to 16 bits once)
//   out[t] = sum over e in S[t] of D_e h[t, e]                                  (fp32, rounded once)
//
// (The routing weight goes into h before its one rounding, so the down product of all experts of a token is
// a single sum in the accumulators.)
//
// Bound by memory: every chosen expert's 3 H I weights are read once and used for a handful of
// tokens. So the weights go straight from global memory to registers in the shape of an MMA's A
// operand (16 weight rows), the tokens ride on its N (8 at a time), and what decides is the bytes in
// flight: a warp has 16 rows x 512 bytes on the way at once, a CTA eight warps that share the rows and split the
// contraction; their sums are joined in shared memory in a fixed order. mma.sync is used because its
// operands are registers: the tensor cores are idle most of the time either way, and a detour of the
// weights through shared and tensor memory would only add latency. Which k an MMA's lanes hold is free as long as
// both operands agree, so a lane takes 16 contiguous bytes of a row and feeds two MMAs with them.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "mx_format.cuh"
#include "ptx.cuh"

namespace b200 {

static constexpr int kMoeMaxTokens = 64;
static constexpr int kMoeMaxExperts = 512;
static constexpr int kMoeMaxTopK = 32;
static constexpr int kMoeThreads = 256;
static constexpr int kMoeWarps = kMoeThreads / 32;
static constexpr int kMoeStep = 256;         // elements of the contraction one warp takes at a time
static constexpr int kRouterCluster = 8;
static constexpr int kRouterTokens = 4;      // tokens one cluster routes

enum MoeWeights : int { kMoe16 = 0, kMoeMxfp4 = 1, kMoeNvfp4 = 2 };

// One product's weights, all experts' rows one below the other.
struct MoeMatrix {
  const uint8_t* data;     // 16-bit values, or codes
  const uint8_t* scales;   // block scales of codes
  long long pitch;         // bytes of a row
  long long col_tiles;     // scale tiles along a row
};

struct MoeArgs {
  int T, E, k, H, I;
  int renormalize;
  const uint16_t* x;        // [T, H]
  const uint16_t* router;   // [E, H]
  const float* bias;        // [E] or NULL
  MoeMatrix w1;             // [E, 2 I, H]: gate rows, then up rows
  MoeMatrix w2;             // [E, H, I]
  float lift1, lift2;       // what sums of products with w1 / w2 are multiplied with (1 for 16-bit weights)
  int* ids;                 // [T, k], -1 = none
  float* weights;           // [T, k]
  uint16_t* h;              // [T, k, I]
  uint16_t* out;            // [T, H]
};

// ------------------------------------------------------------------------------------- small pieces
// D (16 x 8, fp32) += A (16 x 16) * B (16 x 8), 16-bit operands.
template <int F16>
B200_DEVICE void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  if constexpr (F16) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  } else {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  }
}

template <int F16>
B200_DEVICE float2 unpack16(uint32_t w) {
  if constexpr (F16) {
    return __half22float2(*reinterpret_cast<const __half2*>(&w));
  } else {
    return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u));
  }
}

template <int F16>
B200_DEVICE uint16_t round16(float v) {
  if constexpr (F16) {
    return __half_as_ushort(__float2half_rn(v));
  } else {
    return __bfloat16_as_ushort(__float2bfloat16_rn(v));
  }
}

// ------------------------------------------------------------------------------------- router
// Order-preserving map of a logit to an unsigned number; NaN is the largest, as in a sort.
B200_DEVICE uint32_t logit_key(float v) {
  if (v != v) return 0xFFFFFFFFu;
  const uint32_t b = __float_as_uint(v + 0.0f);  // -0 becomes +0
  return (b & 0x80000000u) ? ~b : b | 0x80000000u;
}
B200_DEVICE float key_logit(uint32_t key) {
  return __uint_as_float((key & 0x80000000u) ? key & 0x7FFFFFFFu : ~key);
}
static constexpr uint32_t kKeyMinusInf = 0x007FFFFFu;  // logit_key(-inf)

// A cluster of 8 CTAs routes up to 4 tokens: CTA r has the experts [E r / 8, E (r + 1) / 8), a warp one expert
// at a time against all tokens of the cluster; the logits of token j go to CTA j, whose first warp chooses.
// Lanes hold the same elements of a dot product whatever T is, so a token's logits do not depend on its company.
template <int F16>
__global__ void __launch_bounds__(kMoeThreads) moe_router_kernel(const __grid_constant__ MoeArgs args) {
  __shared__ float logits[kMoeMaxExperts];
  const int warp = static_cast<int>(threadIdx.x) / 32;
  const int lane = static_cast<int>(threadIdx.x) % 32;
  const int rank = static_cast<int>(ptx::cluster_ctarank());
  const int t0 = static_cast<int>(blockIdx.x) / kRouterCluster * kRouterTokens;
  const int tokens = min(kRouterTokens, args.T - t0);
  ptx::grid_launch_dependents();
  ptx::grid_dependency_wait();
  ptx::cluster_arrive();  // every CTA of the cluster runs before anyone writes into another's shared memory
  ptx::cluster_wait();
  const int e_end = args.E * (rank + 1) / kRouterCluster;
  const uint32_t logits_addr = ptx::smem_u32(logits);
  for (int e = args.E * rank / kRouterCluster + warp; e < e_end; e += kMoeWarps) {
    float acc[kRouterTokens][2] = {};
    const uint16_t* w = args.router + static_cast<long long>(e) * args.H;
#pragma unroll 4
    for (int c = lane * 8; c < args.H; c += 256) {
      const uint4 q = *reinterpret_cast<const uint4*>(w + c);
      const uint32_t qw[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
      for (int j = 0; j < kRouterTokens; ++j) {
        if (j < tokens) {
          const uint4 v = *reinterpret_cast<const uint4*>(args.x + static_cast<long long>(t0 + j) * args.H + c);
          const uint32_t vw[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float2 a = unpack16<F16>(qw[i]), b = unpack16<F16>(vw[i]);
            acc[j][0] = fmaf(a.x, b.x, acc[j][0]);
            acc[j][1] = fmaf(a.y, b.y, acc[j][1]);
          }
        }
      }
    }
    const float bias = args.bias != nullptr ? args.bias[e] : 0.0f;
#pragma unroll
    for (int j = 0; j < kRouterTokens; ++j) {
      float s = acc[j][0] + acc[j][1];
#pragma unroll
      for (int d = 16; d > 0; d >>= 1) s += __shfl_xor_sync(0xFFFFFFFFu, s, d);
      if (lane == 0 && j < tokens) {
        asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(ptx::map_to_cta(logits_addr + e * 4, j)), "f"(s + bias)
                     : "memory");
      }
    }
  }
  __syncwarp();
  ptx::cluster_arrive();
  ptx::cluster_wait();
  if (warp != 0 || rank >= tokens) return;
  const int t = t0 + rank;
  constexpr int kPer = kMoeMaxExperts / 32;
  uint32_t key[kPer];  // experts lane, lane + 32, ...; 0 = none or taken
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int e = i * 32 + lane;
    key[i] = e < args.E ? logit_key(logits[e]) : 0u;
  }
  float mine = 0.0f, sum = 0.0f, top = 0.0f;  // lane j keeps the j-th choice
  int id = -1;
  float total_all = 0.0f;
  for (int j = 0; j < args.k; ++j) {
    uint32_t best = 0u;
#pragma unroll
    for (int i = 0; i < kPer; ++i) best = max(best, key[i]);
    best = __reduce_max_sync(0xFFFFFFFFu, best);
    if (best <= kKeyMinusInf) break;
    uint32_t at = 0xFFFFFFFFu;
#pragma unroll
    for (int i = kPer - 1; i >= 0; --i) {
      if (key[i] == best) at = static_cast<uint32_t>(i * 32 + lane);
    }
    at = __reduce_min_sync(0xFFFFFFFFu, at);
    const float v = best == 0xFFFFFFFFu ? __uint_as_float(0x7FC00000u) : key_logit(best);
    if (j == 0) {
      top = v;
      if (!args.renormalize) {
        float s = 0.0f;
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
          if (i * 32 + lane < args.E) s += expf(logits[i * 32 + lane] - top);
        }
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) s += __shfl_xor_sync(0xFFFFFFFFu, s, d);
        total_all = s;
      }
    }
    const float p = expf(v - top);
    sum += p;
    if (lane == j) {
      mine = p;
      id = static_cast<int>(at);
    }
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      if (static_cast<uint32_t>(i * 32 + lane) == at) key[i] = 0u;
    }
  }
  if (lane < args.k) {
    const float total = args.renormalize ? sum : total_all;
    args.ids[t * args.k + lane] = id;
    args.weights[t * args.k + lane] = id < 0 ? 0.0f : __fdiv_rn(mine, total);
  }
}

// ------------------------------------------------------------------------------------- routing tables
// What a CTA of the two product kernels knows of the routing, built from ids by itself: the experts
// anybody chose, the tokens of each as a bit mask, and the (token, choice) pairs ordered by
// expert and token.
struct RouteTables {
  unsigned long long* mask;  // [E]
  uint16_t* list;            // [E] chosen experts, ascending
  uint16_t* first;           // [E] first pair of an expert in `pairs`
  uint16_t* pairs;           // [T * k] token * k + choice
  int* count;                // chosen experts
};

__host__ __device__ __forceinline__ int route_table_bytes(int E, int pairs) {
  return E * 8 + E * 2 + E * 2 + pairs * 2 + 16 + 16;
}

B200_DEVICE RouteTables route_tables_at(uint8_t* smem, const MoeArgs& args) {
  RouteTables r;
  r.mask = reinterpret_cast<unsigned long long*>(smem);
  r.count = reinterpret_cast<int*>(smem + args.E * 8);
  r.list = reinterpret_cast<uint16_t*>(smem + args.E * 8 + 16);
  r.first = r.list + args.E;
  r.pairs = r.first + args.E;
  return r;
}

B200_DEVICE void build_route_tables(const RouteTables& r, const MoeArgs& args) {
  const int t = static_cast<int>(threadIdx.x);
  const int pairs = args.T * args.k;
  for (int e = t; e < args.E; e += kMoeThreads) r.mask[e] = 0ull;
  __syncthreads();
  for (int p = t; p < pairs; p += kMoeThreads) {
    const int e = __ldcg(args.ids + p);
    if (e >= 0) atomicOr(r.mask + e, 1ull << (p / args.k));
  }
  __syncthreads();
  if (t < 32) {
    int found = 0, base = 0;
    for (int e0 = 0; e0 < args.E; e0 += 32) {
      const int e = e0 + t;
      const int n = e < args.E ? __popcll(r.mask[e]) : 0;
      const uint32_t some = __ballot_sync(0xFFFFFFFFu, n > 0);
      int before = n;  // inclusive prefix of the pair counts
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const int other = __shfl_up_sync(0xFFFFFFFFu, before, d);
        if (t >= d) before += other;
      }
      if (e < args.E) r.first[e] = static_cast<uint16_t>(base + before - n);
      if (n > 0) r.list[found + __popc(some & ((1u << t) - 1u))] = static_cast<uint16_t>(e);
      found += __popc(some);
      base += __shfl_sync(0xFFFFFFFFu, before, 31);
    }
    if (t == 0) *r.count = found;
  }
  __syncthreads();
  for (int p = t; p < pairs; p += kMoeThreads) {
    const int e = __ldcg(args.ids + p);
    if (e >= 0) {
      const unsigned long long lower = r.mask[e] & ((1ull << (p / args.k)) - 1ull);
      r.pairs[r.first[e] + __popcll(lower)] = static_cast<uint16_t>(p);
    }
  }
  __syncthreads();
}

// ------------------------------------------------------------------------------------- weights in registers
// One warp's share of a step: MT x 16 weight rows against kMoeStep elements from k0 on. Row g of MMA m
// is `rows(m, 0)`, row g + 8 is `rows(m, 1)` (negative: zeros). B operands come from `cols(j, &any)`, the vector
// of column g of n-tile j (NULL: zeros; any = false: no column of the tile is in use).
//
// 16-bit weights: eight chunks of 32 elements, a lane 16 bytes of each row and chunk.
template <int F16, int NT, int MT, typename Rows, typename Cols>
B200_DEVICE void weight_step16(float (&acc)[MT][NT][4], const MoeMatrix& w, int k0, int K, uint32_t lane, Rows rows,
                               Cols cols) {
  const int kl = k0 + static_cast<int>(lane & 3u) * 8;
  uint4 q[MT][2][8];
#pragma unroll
  for (int m = 0; m < MT; ++m) {
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      const long long row = rows(m, half);
      const uint8_t* p = w.data + row * w.pitch + kl * 2;
#pragma unroll
      for (int c = 0; c < 8; ++c) {
        q[m][half][c] = (row >= 0 && kl + c * 32 < K) ? ptx::ld_stream_v4(p + c * 64) : make_uint4(0u, 0u, 0u, 0u);
      }
    }
  }
#pragma unroll
  for (int j = 0; j < NT; ++j) {
    bool any;
    const uint16_t* b = cols(j, &any);
    if (!any) continue;  // (the same for the whole warp)
#pragma unroll
    for (int c = 0; c < 8; ++c) {
      const uint4 v = (b != nullptr && kl + c * 32 < K) ? *reinterpret_cast<const uint4*>(b + kl + c * 32)
                                                        : make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
      for (int m = 0; m < MT; ++m) {
        mma16816<F16>(acc[m][j], q[m][0][c].x, q[m][1][c].x, q[m][0][c].y, q[m][1][c].y, v.x, v.y);
        mma16816<F16>(acc[m][j], q[m][0][c].z, q[m][1][c].z, q[m][0][c].w, q[m][1][c].w, v.z, v.w);
      }
    }
  }
}

// What a 4-bit weight's bits are multiplied with. A code's magnitude bits at the top of a bf16 number's mantissa
// and the bottom of its exponent read code * 2^-126; two factors (the second nearly always 1) bring them to
// code * scale (MXFP4) or code * scale * 2^-16 (NVFP4, whose block scales reach 448: the rest is
// applied to the sums). Every product is exact in bf16.
static constexpr float kNvfp4Lift = 65536.0f;
template <int W>
B200_DEVICE void weight_factors(uint32_t byte, uint32_t* first, uint32_t* second) {
  uint32_t f, s = 0x3F80u;
  if constexpr (W == kMoeMxfp4) {
    f = byte == 255u ? 0x7FC0u : min(byte + 126u, 254u) << 7;
    if (byte > 128u) s = (byte - 1u) << 7;  // 2^(byte - 128)
  } else {
    f = __float_as_uint(e4m3_value(byte) * 1.298074214633707e33f) >> 16;  // 2^110
  }
  *first = f | (f << 16);
  *second = s | (s << 16);
}

B200_DEVICE uint32_t mul_bf16x2(uint32_t a, uint32_t b) {
  uint32_t d;
  asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}

// 4-bit weights: two chunks of 128 elements, a lane 16 bytes = 32 elements of each row and chunk. Of a word's
// eight codes, i and i + 4 are 16 bits apart: one shift brings both to their place in a bf16 pair, and B
// takes its elements in the same order.
template <int W, int NT, int MT, typename Rows, typename Cols>
B200_DEVICE void weight_step4(float (&acc)[MT][NT][4], const MoeMatrix& w, int k0, int K, uint32_t lane, Rows rows,
                              Cols cols) {
  constexpr int FMT = W == kMoeMxfp4 ? kMxfp4 : kNvfp4;
  constexpr int kBlocks = 32 / mx_block(FMT);  // block scales of a lane's 32 elements
  const int part = static_cast<int>(lane & 3u);
  uint4 q[MT][2][2];
  uint32_t sb[MT][2][2];
#pragma unroll
  for (int m = 0; m < MT; ++m) {
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      const long long row = rows(m, half);
      const uint8_t* p = w.data + row * w.pitch + k0 / 2 + part * 16;
      const uint8_t* sp = w.scales + mx_scale_offset(FMT, row, k0 / mx_block(FMT) + part * kBlocks, w.col_tiles);
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const bool live = row >= 0 && k0 + c * 128 + part * 32 < K;
        q[m][half][c] = live ? ptx::ld_stream_v4(p + c * 64) : make_uint4(0u, 0u, 0u, 0u);
        sb[m][half][c] = 0u;
        if (live) {
          if constexpr (FMT == kMxfp4) {
            sb[m][half][c] = sp[c * kMxGroupBytes];
          } else {
            sb[m][half][c] = *reinterpret_cast<const uint16_t*>(sp + c * 2 * kMxGroupBytes);
          }
        }
      }
    }
  }
#pragma unroll
  for (int c = 0; c < 2; ++c) {
#pragma unroll
    for (int word = 0; word < 4; ++word) {
      const int k = k0 + c * 128 + part * 32 + word * 8;
      uint32_t a[MT][2][4];
#pragma unroll
      for (int m = 0; m < MT; ++m) {
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const uint4& v = q[m][half][c];
          const uint32_t codes = word == 0 ? v.x : word == 1 ? v.y : word == 2 ? v.z : v.w;
          uint32_t f, s;
          weight_factors<W>((sb[m][half][c] >> (kBlocks == 2 ? (word / 2) * 8 : 0)) & 0xFFu, &f, &s);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const uint32_t mag = (i < 2 ? codes << (6 - 4 * i) : codes >> (4 * i - 6)) & 0x01C001C0u;
            const uint32_t bits = mag | ((codes << (12 - 4 * i)) & 0x80008000u);
            uint32_t d = mul_bf16x2(bits, f);
            if constexpr (W == kMoeMxfp4) d = mul_bf16x2(d, s);
            a[m][half][i] = d;
          }
        }
      }
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        bool any;
        const uint16_t* b = cols(j, &any);
        if (!any) continue;
        const uint4 v = (b != nullptr && k < K) ? *reinterpret_cast<const uint4*>(b + k) : make_uint4(0u, 0u, 0u, 0u);
        const uint32_t b0 = __byte_perm(v.x, v.z, 0x5410), b1 = __byte_perm(v.x, v.z, 0x7632);
        const uint32_t b2 = __byte_perm(v.y, v.w, 0x5410), b3 = __byte_perm(v.y, v.w, 0x7632);
#pragma unroll
        for (int m = 0; m < MT; ++m) {
          mma16816<0>(acc[m][j], a[m][0][0], a[m][1][0], a[m][0][1], a[m][1][1], b0, b1);
          mma16816<0>(acc[m][j], a[m][0][2], a[m][1][2], a[m][0][3], a[m][1][3], b2, b3);
        }
      }
    }
  }
}

template <int W, int F16, int NT, int MT, typename Rows, typename Cols>
B200_DEVICE void weight_step(float (&acc)[MT][NT][4], const MoeMatrix& w, int k0, int K, uint32_t lane, Rows rows,
                             Cols cols) {
  if constexpr (W == kMoe16) {
    weight_step16<F16, NT, MT>(acc, w, k0, K, lane, rows, cols);
  } else {
    weight_step4<W, NT, MT>(acc, w, k0, K, lane, rows, cols);
  }
}

// MMA tiles of weight rows a unit has: 4-bit rows are a quarter as long, so a unit takes two to keep as much on the way.
template <int W>
struct MoeUnit {
  static constexpr int kTiles = W == kMoe16 ? 1 : 2;
  static constexpr float kLift = W == kMoeNvfp4 ? kNvfp4Lift : 1.0f;
};

B200_DEVICE float silu(float v) { return __fdividef(v, 1.0f + __expf(-v)); }

// ------------------------------------------------------------------------------------- gate and up
// Unit: 8 intermediate columns per MMA tile of one chosen expert = 8 gate rows and the 8 up rows beside them, so that
// a lane ends up with a gate value and its up value. The CTAs take units in turn.
template <int W, int F16, int NT>
B200_DEVICE void gate_up_unit(const MoeArgs& args, const RouteTables& r, float4* red, int e, int i0, int tokens) {
  constexpr int MT = MoeUnit<W>::kTiles;
  const uint32_t lane = ptx::lane_id();
  const int warp = static_cast<int>(threadIdx.x) / 32;
  const int g = static_cast<int>(lane >> 2);
  const uint16_t* pairs = r.pairs + r.first[e];
  const uint16_t* xrow[NT];
#pragma unroll
  for (int j = 0; j < NT; ++j) {
    xrow[j] = j * 8 + g < tokens ? args.x + static_cast<long long>(pairs[j * 8 + g] / args.k) * args.H : nullptr;
  }
  const long long row0 = static_cast<long long>(e) * 2 * args.I + i0 + g;
  float acc[MT][NT][4] = {};
  for (int k0 = warp * kMoeStep; k0 < args.H; k0 += kMoeWarps * kMoeStep) {
    weight_step<W, F16, NT, MT>(
        acc, args.w1, k0, args.H, lane,
        [&](int m, int half) { return i0 + m * 8 < args.I ? row0 + m * 8 + (half ? args.I : 0) : -1ll; },
        [&](int j, bool* any) {
          *any = j * 8 < tokens;
          return xrow[j];
        });
  }
#pragma unroll
  for (int m = 0; m < MT; ++m) {
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      red[((warp * MT + m) * NT + j) * 32 + lane] = make_float4(acc[m][j][0], acc[m][j][1], acc[m][j][2], acc[m][j][3]);
    }
  }
  __syncthreads();
  for (int idx = static_cast<int>(threadIdx.x); idx < MT * NT * 32; idx += kMoeThreads) {
    float4 s = red[idx];
#pragma unroll
    for (int p = 1; p < kMoeWarps; ++p) {
      const float4 v = red[p * MT * NT * 32 + idx];
      s.x += v.x;
      s.y += v.y;
      s.z += v.z;
      s.w += v.w;
    }
    const int tile = idx / 32;
    const int row = i0 + tile / NT * 8 + (idx % 32) / 4;
    const int c = tile % NT * 8 + (idx % 4) * 2;
    const float gate[2] = {s.x, s.y}, up[2] = {s.z, s.w};
    if (row >= args.I) continue;
#pragma unroll
    for (int n = 0; n < 2; ++n) {
      if (c + n < tokens) {
        const int pair = pairs[c + n];
        const float p = __ldcg(args.weights + pair);
        args.h[static_cast<long long>(pair) * args.I + row] = round16<F16>(p * (silu(gate[n] * args.lift1) * (up[n] * args.lift1)));
      }
    }
  }
}

__host__ __device__ __forceinline__ int moe_token_tiles(int T) { return T <= 8 ? 1 : T <= 16 ? 2 : T <= 32 ? 4 : 8; }

template <int W, int F16>
__global__ void __launch_bounds__(kMoeThreads, 2) moe_gate_up_kernel(const __grid_constant__ MoeArgs args) {
  constexpr int kCols = 8 * MoeUnit<W>::kTiles;
  extern __shared__ __align__(16) uint8_t smem[];
  float4* red = reinterpret_cast<float4*>(smem);  // two buffers, used in turn
  const int red_bytes = kMoeWarps * 32 * 16 * MoeUnit<W>::kTiles * moe_token_tiles(args.T);
  const RouteTables r = route_tables_at(smem + 2 * red_bytes, args);
  ptx::grid_launch_dependents();
  ptx::grid_dependency_wait();
  build_route_tables(r, args);
  const int strips = (args.I + kCols - 1) / kCols;
  const int units = *r.count * strips;
  int turn = 0;
  for (int u = static_cast<int>(blockIdx.x); u < units; u += static_cast<int>(gridDim.x), turn ^= 1) {
    const int e = r.list[u / strips];
    const int i0 = u % strips * kCols;
    const int tokens = __popcll(r.mask[e]);
    float4* buffer = red + turn * (red_bytes / 16);
    if (tokens <= 8) {
      gate_up_unit<W, F16, 1>(args, r, buffer, e, i0, tokens);
    } else if (tokens <= 16) {
      gate_up_unit<W, F16, 2>(args, r, buffer, e, i0, tokens);
    } else if (tokens <= 32) {
      gate_up_unit<W, F16, 4>(args, r, buffer, e, i0, tokens);
    } else {
      gate_up_unit<W, F16, 8>(args, r, buffer, e, i0, tokens);
    }
  }
}

// ------------------------------------------------------------------------------------- down
// Unit: 16 columns of the output per MMA tile, for all tokens, one cluster. The contraction runs over all
// chosen experts; its steps go to the warps of the cluster in turn. Column g of n-tile j is token 8 j + g for every
// expert (zeros where it did not choose it), so the accumulators add the experts up by themselves.
template <int W, int F16, int NT>
__global__ void __launch_bounds__(kMoeThreads, 2) moe_down_kernel(const __grid_constant__ MoeArgs args, int split) {
  constexpr int MT = MoeUnit<W>::kTiles;
  extern __shared__ __align__(16) uint8_t smem[];
  float4* red = reinterpret_cast<float4*>(smem);
  const RouteTables r = route_tables_at(smem + kMoeWarps * MT * NT * 32 * 16, args);
  const uint32_t lane = ptx::lane_id();
  const int warp = static_cast<int>(threadIdx.x) / 32;
  const int rank = split > 1 ? static_cast<int>(ptx::cluster_ctarank()) : 0;
  const int r0 = static_cast<int>(blockIdx.x) / split * 16 * MT;
  const int g = static_cast<int>(lane >> 2);
  ptx::grid_launch_dependents();
  ptx::grid_dependency_wait();
  build_route_tables(r, args);
  const int steps = (args.I + kMoeStep - 1) / kMoeStep;
  const int total = *r.count * steps;
  float acc[MT][NT][4] = {};
  for (int s = rank * kMoeWarps + warp; s < total; s += split * kMoeWarps) {
    const int e = r.list[s / steps];
    const unsigned long long mask = r.mask[e];
    const uint16_t* pairs = r.pairs + r.first[e];
    weight_step<W, F16, NT, MT>(
        acc, args.w2, s % steps * kMoeStep, args.I, lane,
        [&](int m, int half) {
          const int row = r0 + m * 16 + half * 8 + g;
          return row < args.H ? static_cast<long long>(e) * args.H + row : -1ll;
        },
        [&](int j, bool* any) -> const uint16_t* {
          *any = ((mask >> (8 * j)) & 0xFFull) != 0;
          const int t = 8 * j + g;
          if (!((mask >> t) & 1ull)) return nullptr;
          const int pair = pairs[__popcll(mask & ((1ull << t) - 1ull))];
          return args.h + static_cast<long long>(pair) * args.I;
        });
  }
#pragma unroll
  for (int m = 0; m < MT; ++m) {
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      red[((warp * MT + m) * NT + j) * 32 + lane] = make_float4(acc[m][j][0], acc[m][j][1], acc[m][j][2], acc[m][j][3]);
    }
  }
  __syncthreads();
  if (split > 1) {
    ptx::cluster_arrive();
    ptx::cluster_wait();
  }
  // CTA `rank` finishes its share of the tiles' elements.
  const uint32_t red_addr = ptx::smem_u32(red);
  for (int idx = rank * kMoeThreads + static_cast<int>(threadIdx.x); idx < MT * NT * 32; idx += split * kMoeThreads) {
    float4 s = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    for (int p = 0; p < split; ++p) {
      const uint32_t base = split > 1 ? ptx::map_to_cta(red_addr, static_cast<uint32_t>(p)) : red_addr;
      for (int q = 0; q < kMoeWarps; ++q) {
        const float4 v = ptx::ld_cluster_v4(base + static_cast<uint32_t>((q * MT * NT * 32 + idx) * 16));
        s.x += v.x;
        s.y += v.y;
        s.z += v.z;
        s.w += v.w;
      }
    }
    const int tile = idx / 32;
    const int row = r0 + tile / NT * 16 + (idx % 32) / 4;
    const int t = tile % NT * 8 + (idx % 4) * 2;
    const float lo[2] = {s.x, s.y}, hi[2] = {s.z, s.w};
#pragma unroll
    for (int n = 0; n < 2; ++n) {
      if (t + n < args.T) {
        uint16_t* o = args.out + static_cast<long long>(t + n) * args.H + row;
        if (row < args.H) o[0] = round16<F16>(lo[n] * args.lift2);
        if (row + 8 < args.H) o[8] = round16<F16>(hi[n] * args.lift2);
      }
    }
  }
  if (split > 1) {
    ptx::cluster_arrive();  // no CTA leaves while another reads its sums
    ptx::cluster_wait();
  }
}

}  // namespace b200
