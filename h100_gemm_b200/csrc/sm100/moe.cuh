// A mixture-of-experts layer for a few tokens (T <= 64), in three kernels of one launch sequence.
//
//   logits  l[t, e] = x[t] . R[e] + b[e]                                        (fp32)
//   chosen  S[t] = the k largest logits of t (ties: the lower index; -inf is never chosen)
//   weight  p[t, e] = exp(l[t, e]) / sum of exp(l) over S[t], or over all experts
//   gated   h[t, e] = p[t, e] * silu(G_e x[t]) * (U_e x[t])                     (fp32)
//   out[t] = sum over e in S[t] of D_e h[t, e]                                  (fp32, rounded once)
//
// (The routing weight goes into h, so the down product of all experts of a token is a single sum. The tensor cores take
// 16-bit operands, so h meets the down weights in parts (HiddenParts), 22 bits of it for bf16: outputs then differ from
// those of an fp32 hidden value as seldom as fp32 sums in another order do.)
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
static constexpr int kRouterCluster = 8;
static constexpr int kRouterThreads = 512;  // at most
static constexpr int kRouterTokens = 4;      // tokens one cluster routes, at most

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
  float scale1[2], scale2[2];  // two factors each of what sums of products with w1 / w2 are multiplied with
  int* ids;                 // [T, k], -1 = none
  float* weights;           // [T, k]
  uint16_t* h;              // [T, k, 2, I]: HiddenParts
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
B200_DEVICE float widen16(uint16_t bits) {
  if constexpr (F16) {
    return __half2float(__ushort_as_half(bits));
  } else {
    return __uint_as_float(static_cast<uint32_t>(bits) << 16);
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

B200_DEVICE uint32_t mul_bf16x2(uint32_t a, uint32_t b) {
  uint32_t d;
  asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}

B200_DEVICE uint32_t sub_bf16x2(uint32_t a, uint32_t b) {
  uint32_t d;
  asm("sub.rn.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}

// ------------------------------------------------------------------------------------- hidden values
// A hidden value takes two 16-bit words, in two planes, and meets the weights in kParts operands whose sums are scaled and
// added. Its elements lie in the order that the weights' MMA takes them in (hidden_place).
//
// bf16: the fp32 number, rounded to 22 significant bits: its upper half, and the next two groups of 7 bits, m1 below m2. With
// E = +-2^e, sign and exponent alone, the parts are the upper half itself, E * m1 / 128 and E * m2 / 128: each
// exact in bf16 and two or three instructions for two elements (E | m is E + E m / 128).
// fp16: the nearest fp16 number, and the nearest one of 2^11 times what that leaves, which is at most 2^15 (half a step of
// the largest numbers) and, unscaled, would be subnormal for hidden values below a quarter. 22 bits from 2^-14 on, 2^-36 below.
template <int F16>
struct HiddenParts;

template <>
struct HiddenParts<0> {
  static constexpr int kParts = 3;
  static B200_DEVICE float factor(int p) { return p == 0 ? 1.0f : p == 1 ? 0.0078125f : 0.00006103515625f; }  // 1, 2^-7, 2^-14
  static B200_DEVICE void store(float h, uint16_t* first, uint16_t* second) {
    const uint32_t bits = h == h ? __float_as_uint(h) + 2u : 0x7FC00000u;  // (beyond the largest number: infinity)
    *first = static_cast<uint16_t>(bits >> 16);
    *second = static_cast<uint16_t>((bits >> 9 & 0x7Fu) | (bits >> 2 & 0x7Fu) << 8);
  }
  static B200_DEVICE uint32_t lower(uint32_t first, uint32_t m) {
    const uint32_t e = first & 0xFF80FF80u;
    return sub_bf16x2((m & 0x007F007Fu) | e, e);
  }
  static B200_DEVICE void all(uint32_t (&part)[kParts], uint32_t first, uint32_t second) {
    part[0] = first;
    part[1] = lower(first, second);
    part[2] = lower(first, second >> 8);
  }
  // Part `p`, the same for all elements of a lane.
  static constexpr int kReads = 2;
  static B200_DEVICE uint32_t one(const uint32_t (&word)[kReads], int p) {
    const uint32_t v = lower(word[0], word[1] >> (p == 2 ? 8 : 0));
    return p == 0 ? word[0] : v;
  }
};

template <>
struct HiddenParts<1> {
  static constexpr int kParts = 2;
  static B200_DEVICE float factor(int p) { return p == 0 ? 1.0f : 0.00048828125f; }  // 1, 2^-11
  static B200_DEVICE void store(float h, uint16_t* first, uint16_t* second) {
    *first = round16<1>(h);
    // (beyond the type's range h becomes infinite, as it would in one part, and not the NaN of inf - inf)
    const float rest = (h - widen16<1>(*first)) * 2048.0f;
    *second = round16<1>(isinf(rest) || isinf(h) ? 0.0f : rest);
  }
  static B200_DEVICE void all(uint32_t (&part)[kParts], uint32_t first, uint32_t second) {
    part[0] = first;
    part[1] = second;
  }
  static constexpr int kReads = 1;  // of the part's own plane
  static B200_DEVICE uint32_t one(const uint32_t (&word)[kReads], int) { return word[0]; }
};

// How the columns of an MMA take hidden vectors (`base`: the first plane, `plane` elements before the second).
// HiddenSums: column g is a token, its parts go to kSums accumulators one after the other. HiddenColumns: the parts of a token
// lie side by side on kWidth columns (of bf16's four one is idle), with one accumulator and a third of the MMAs. An expert
// with as few tokens as one tile of those holds takes them: 4 tokens 54.2 us against 57.8 with sums alone, 16 tokens
// 123.4 against 130, 4 tokens MXFP4 40.3 against 43. (Two such tiles at once for 3 and 4 tokens: 16 tokens 122 us, but 64
// tokens of 4-bit experts 176 against 155, a third variant of the unrolled product being too much code.)
template <int F16>
struct HiddenSums {
  using P = HiddenParts<F16>;
  static constexpr int kSums = P::kParts, kReads = 2, kTokens = 8;
  const uint16_t* at[kReads];
  B200_DEVICE HiddenSums(const uint16_t* base, int plane, int) : at{base, base + plane} {}
  B200_DEVICE void operands(uint32_t (&b)[kSums][4], const uint4 (&v)[kReads]) const {
    const uint32_t first[4] = {v[0].x, v[0].y, v[0].z, v[0].w}, second[4] = {v[1].x, v[1].y, v[1].z, v[1].w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      uint32_t part[kSums];
      P::all(part, first[i], second[i]);
#pragma unroll
      for (int p = 0; p < kSums; ++p) b[p][i] = part[p];
    }
  }
};

template <int F16>
struct HiddenColumns {
  using P = HiddenParts<F16>;
  static constexpr int kWidth = P::kParts == 3 ? 4 : 2;
  static constexpr int kSums = 1, kReads = P::kReads, kTokens = 8 / kWidth;
  const uint16_t* at[kReads];
  int part;
  B200_DEVICE HiddenColumns(const uint16_t* base, int plane, int column) : part(column % kWidth) {
    at[0] = kReads == 1 ? base + part * plane : base;
    if constexpr (kReads == 2) at[1] = base + plane;
  }
  B200_DEVICE void operands(uint32_t (&b)[1][4], const uint4 (&v)[kReads]) const {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      uint32_t word[kReads];
#pragma unroll
      for (int r = 0; r < kReads; ++r) word[r] = i == 0 ? v[r].x : i == 1 ? v[r].y : i == 2 ? v[r].z : v[r].w;
      b[0][i] = P::one(word, part);
    }
  }
};

// The parts' sums as one. Where an infinite or NaN hidden value makes the first sum that, the others hold inf - inf: the first
// alone is what the formula gives.
template <int F16>
B200_DEVICE float join_parts(const float (&sum)[HiddenParts<F16>::kParts]) {
  float v = sum[0];
#pragma unroll
  for (int p = 1; p < HiddenParts<F16>::kParts; ++p) v = fmaf(sum[p], HiddenParts<F16>::factor(p), v);
  return isfinite(sum[0]) ? v : sum[0];
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

// A cluster of 8 CTAs routes TOKENS tokens: CTA r has the experts [E r / 8, E (r + 1) / 8), a warp one expert
// at a time against all tokens of the cluster; the logits of token j go to CTA j, whose first warp chooses.
// Bound by latency, so the loads of 1024 elements of every row are on the way together (with a branch
// around each token's loads, 4 tokens of 2048 and 128 experts took 29 us; now 6). Lanes hold the same elements of a
// dot product whatever T is, so a token's logits do not depend on its company.
template <int F16, int TOKENS>
__global__ void __launch_bounds__(kRouterThreads) moe_router_kernel(const __grid_constant__ MoeArgs args) {
  __shared__ float logits[kMoeMaxExperts];
  const int warp = static_cast<int>(threadIdx.x) / 32;
  const int lane = static_cast<int>(threadIdx.x) % 32;
  const int rank = static_cast<int>(ptx::cluster_ctarank());
  const int t0 = static_cast<int>(blockIdx.x) / kRouterCluster * TOKENS;
  const int tokens = min(TOKENS, args.T - t0);
  ptx::grid_launch_dependents();
  ptx::cluster_arrive();  // every CTA of the cluster runs before anyone writes into another's shared memory
  ptx::cluster_wait();
  ptx::grid_dependency_wait();
  const int e_end = args.E * (rank + 1) / kRouterCluster;
  const uint32_t logits_addr = ptx::smem_u32(logits);
  const uint16_t* xrow[TOKENS];
#pragma unroll
  for (int j = 0; j < TOKENS; ++j) xrow[j] = args.x + static_cast<long long>(min(t0 + j, args.T - 1)) * args.H;
  for (int e = args.E * rank / kRouterCluster + warp; e < e_end; e += static_cast<int>(blockDim.x) / 32) {
    float acc[TOKENS][2] = {};
    const uint16_t* w = args.router + static_cast<long long>(e) * args.H;
    for (int base = 0; base < args.H; base += 1024) {
      uint4 q[4], v[TOKENS][4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        // (beyond the row: its last elements again, not used)
        const int c = base + i * 256 + lane * 8;
        const int at = min(c, args.H - 8);
        q[i] = *reinterpret_cast<const uint4*>(w + at);
#pragma unroll
        for (int j = 0; j < TOKENS; ++j) v[j][i] = *reinterpret_cast<const uint4*>(xrow[j] + at);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (base + i * 256 + lane * 8 >= args.H) continue;
        const uint32_t qw[4] = {q[i].x, q[i].y, q[i].z, q[i].w};
#pragma unroll
        for (int j = 0; j < TOKENS; ++j) {
          const uint32_t vw[4] = {v[j][i].x, v[j][i].y, v[j][i].z, v[j][i].w};
#pragma unroll
          for (int h = 0; h < 4; ++h) {
            const float2 a = unpack16<F16>(qw[h]), b = unpack16<F16>(vw[h]);
            acc[j][0] = fmaf(a.x, b.x, acc[j][0]);
            acc[j][1] = fmaf(a.y, b.y, acc[j][1]);
          }
        }
      }
    }
    const float bias = args.bias != nullptr ? args.bias[e] : 0.0f;
#pragma unroll
    for (int j = 0; j < TOKENS; ++j) {
      float s = acc[j][0] + acc[j][1];
#pragma unroll
      for (int d = 16; d > 0; d >>= 1) s += __shfl_xor_sync(0xFFFFFFFFu, s, d);
      if (lane == 0 && j < tokens) {
        // (an expert that is masked out stays out, whatever its product is: NaN + -inf would be a NaN, the first choice)
        asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(ptx::map_to_cta(logits_addr + e * 4, j)),
                     "f"(bias == -INFINITY ? bias : s + bias)
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
// anybody chose in ascending order, and the (token, choice) pairs ordered by expert and token.
struct RouteTables {
  unsigned long long* mask;  // [E] tokens of an expert (while the tables are built)
  float* weights;            // routing weight of a pair
  int* count;                // chosen experts
  uint16_t* pairs;           // [T * k] token * k + choice
  uint16_t* list;            // [E] chosen experts
  uint16_t* first;           // [E] their first pairs (while the tables are built: by expert)
  uint8_t* tokens;           // token of a pair
  uint8_t* size;             // [E] tokens of a chosen expert
};

__host__ __device__ __forceinline__ int route_table_bytes(int E, int pairs) { return (E * 13 + pairs * 7 + 16 + 15) / 16 * 16; }

B200_DEVICE RouteTables route_tables_at(uint8_t* smem, const MoeArgs& args) {
  const int pairs = args.T * args.k;
  RouteTables r;
  r.mask = reinterpret_cast<unsigned long long*>(smem);
  r.weights = reinterpret_cast<float*>(r.mask + args.E);
  r.count = reinterpret_cast<int*>(r.weights + pairs);
  r.pairs = reinterpret_cast<uint16_t*>(r.count + 1);
  r.list = r.pairs + pairs;
  r.first = r.list + args.E;
  r.tokens = reinterpret_cast<uint8_t*>(r.first + args.E);
  r.size = r.tokens + pairs;
  return r;
}

// Up to 32 pairs, a decode step of one to a few tokens: one warp, a lane a pair, every lane compared with every other.
B200_DEVICE void build_small_route_tables(const RouteTables& r, const MoeArgs& args) {
  const int lane = static_cast<int>(threadIdx.x);
  if (lane < 32) {
    const int pairs = args.T * args.k;
    const int e = lane < pairs ? __ldcg(args.ids + lane) : -1;
    const float weight = e >= 0 ? __ldcg(args.weights + lane) : 0.0f;
    int before = 0, same = 0, same_before = 0;
    for (int q = 0; q < pairs; ++q) {
      const int other = __shfl_sync(0xFFFFFFFFu, e, q);
      before += other >= 0 && other < e;
      same += other == e;
      same_before += other == e && q < lane;
    }
    const bool head = e >= 0 && same_before == 0;
    int index = 0;  // chosen experts before this one
    for (int q = 0; q < pairs; ++q) {
      const int other = __shfl_sync(0xFFFFFFFFu, head ? e : 0x7FFFFFFF, q);
      index += other < e;
    }
    if (e >= 0) {
      r.pairs[before + same_before] = static_cast<uint16_t>(lane);
      r.tokens[before + same_before] = static_cast<uint8_t>(lane / args.k);
      r.weights[before + same_before] = weight;
    }
    if (head) {
      r.list[index] = static_cast<uint16_t>(e);
      r.first[index] = static_cast<uint16_t>(before);
      r.size[index] = static_cast<uint8_t>(same);
    }
    const uint32_t heads = __ballot_sync(0xFFFFFFFFu, head);
    if (lane == 0) *r.count = __popc(heads);
  }
  __syncthreads();
}

B200_DEVICE void build_route_tables(const RouteTables& r, const MoeArgs& args) {
  const int t = static_cast<int>(threadIdx.x);
  const int pairs = args.T * args.k;
  if (pairs <= 32) {
    build_small_route_tables(r, args);
    return;
  }
  constexpr int kPer = kMoeMaxTokens * kMoeMaxTopK / kMoeThreads;  // pairs of a thread, kept for the second pass
  int mine[kPer];
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int p = t + i * kMoeThreads;
    mine[i] = p < pairs ? __ldcg(args.ids + p) : -1;
  }
  for (int e = t; e < args.E; e += kMoeThreads) r.mask[e] = 0ull;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    if (mine[i] >= 0) atomicOr(r.mask + mine[i], 1ull << ((t + i * kMoeThreads) / args.k));
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
      if (n > 0) {
        const int index = found + __popc(some & ((1u << t) - 1u));
        r.list[index] = static_cast<uint16_t>(e);
        r.size[index] = static_cast<uint8_t>(n);
      }
      found += __popc(some);
      base += __shfl_sync(0xFFFFFFFFu, before, 31);
    }
    if (t == 0) *r.count = found;
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int e = mine[i], p = t + i * kMoeThreads;
    if (e >= 0) {
      const int token = p / args.k;
      const int at = r.first[e] + __popcll(r.mask[e] & ((1ull << token) - 1ull));
      r.pairs[at] = static_cast<uint16_t>(p);
      r.tokens[at] = static_cast<uint8_t>(token);
      r.weights[at] = __ldcg(args.weights + p);
    }
  }
  __syncthreads();
  // From by expert to by position: position i's expert is not before i, so going up overwrites nothing still to be read.
  if (t < 32) {
    for (int i0 = 0; i0 < *r.count; i0 += 32) {
      const int i = i0 + t;
      const uint16_t first = i < *r.count ? r.first[r.list[i]] : 0;
      __syncwarp();
      if (i < *r.count) r.first[i] = first;
      __syncwarp();
    }
  }
  __syncthreads();
}

// ------------------------------------------------------------------------------------- weights in registers
// One warp's share of a step: MT x 16 weight rows against kStep elements of the contraction from k0 on. Row g of MMA m
// is `rows(m, 0)`, row g + 8 is `rows(m, 1)` (negative: zeros). load() only issues the loads; mma_tokens() multiplies
// with n-tiles whose column g is the vector `b[j]`, mma_hidden() with one of hidden values.
//
// 16-bit weights: CHUNKS times 32 elements, a lane 16 bytes of each row and chunk.
template <int F16, int MT, int CHUNKS>
struct WeightStep {
  static constexpr int kStep = CHUNKS * 32;
  uint4 q[MT][2][CHUNKS];

  template <typename Rows>
  B200_DEVICE void load(const MoeMatrix& w, int k0, int K, uint32_t lane, Rows rows) {
    const int kl = k0 + static_cast<int>(lane & 3u) * 8;
#pragma unroll
    for (int m = 0; m < MT; ++m) {
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const int row = rows(m, half);
        const uint8_t* p = w.data + row * w.pitch + kl * 2;
        if (row >= 0 && k0 + kStep <= K) {
#pragma unroll
          for (int c = 0; c < CHUNKS; ++c) q[m][half][c] = ptx::ld_stream_v4(p + c * 64);
        } else {
#pragma unroll
          for (int c = 0; c < CHUNKS; ++c) {
            q[m][half][c] = make_uint4(0u, 0u, 0u, 0u);
            if (row >= 0 && kl + c * 32 < K) q[m][half][c] = ptx::ld_stream_v4(p + c * 64);
          }
        }
      }
    }
  }

  B200_DEVICE void mma(float (&acc)[MT][4], const uint16_t* b, int k0, int K, uint32_t lane) const {
    const int kl = k0 + static_cast<int>(lane & 3u) * 8;
#pragma unroll
    for (int c0 = 0; c0 < CHUNKS; c0 += 4) {  // (eight at once would spill)
      uint4 v[4];
      if (k0 + kStep <= K) {
#pragma unroll
        for (int c = 0; c < 4; ++c) v[c] = *reinterpret_cast<const uint4*>(b + kl + (c0 + c) * 32);
      } else {
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          v[c] = make_uint4(0u, 0u, 0u, 0u);
          if (kl + (c0 + c) * 32 < K) v[c] = *reinterpret_cast<const uint4*>(b + kl + (c0 + c) * 32);
        }
      }
#pragma unroll
      for (int c = 0; c < 4; ++c) {
#pragma unroll
        for (int m = 0; m < MT; ++m) {
          const uint4 &lo = q[m][0][c0 + c], &hi = q[m][1][c0 + c];
          mma16816<F16>(acc[m], lo.x, hi.x, lo.y, hi.y, v[c].x, v[c].y);
          mma16816<F16>(acc[m], lo.z, hi.z, lo.w, hi.w, v[c].z, v[c].w);
        }
      }
    }
  }

  template <int NT>
  B200_DEVICE void mma_tokens(float (&acc)[NT][MT][4], const uint16_t* const (&b)[NT], int k0, int K, uint32_t lane) const {
#pragma unroll
    for (int j = 0; j < NT; ++j) mma(acc[j], b[j], k0, K, lane);
  }

  static B200_DEVICE int hidden_place(int i) { return i; }
  template <typename Hidden>
  B200_DEVICE void mma_hidden(float (&acc)[Hidden::kSums][MT][4], const Hidden& columns, int k0, int K, uint32_t lane) const {
    const int kl = k0 + static_cast<int>(lane & 3u) * 8;
#pragma unroll
    for (int c0 = 0; c0 < CHUNKS; c0 += 2) {
      uint4 v[2][Hidden::kReads];
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const int at = kl + (c0 + c) * 32;
#pragma unroll
        for (int r = 0; r < Hidden::kReads; ++r) {
          v[c][r] = make_uint4(0u, 0u, 0u, 0u);
          if (k0 + kStep <= K || at < K) v[c][r] = *reinterpret_cast<const uint4*>(columns.at[r] + at);
        }
      }
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        uint32_t b[Hidden::kSums][4];
        columns.operands(b, v[c]);
#pragma unroll
        for (int j = 0; j < Hidden::kSums; ++j) {
#pragma unroll
          for (int m = 0; m < MT; ++m) {
            const uint4 &lo = q[m][0][c0 + c], &hi = q[m][1][c0 + c];
            mma16816<F16>(acc[j][m], lo.x, hi.x, lo.y, hi.y, b[j][0], b[j][1]);
            mma16816<F16>(acc[j][m], lo.z, hi.z, lo.w, hi.w, b[j][2], b[j][3]);
          }
        }
      }
    }
  }
};

// 4-bit weights: CHUNKS times 128 elements, a lane 16 bytes = 32 elements of each row and chunk.
//
// Unpacking, not memory, is what these kernels spend most instructions on (and waits for their fetch: of a down kernel's
// stalled cycles more than a quarter). A code's magnitude bits at the top of a
// bf16 number's mantissa and the bottom of its exponent read code * 2^-126. Of a word's eight codes, i and
// i + 4 are 16 bits apart, so a mask, one multiplication (which puts the magnitude at bit 6 and the sign
// at bit 15 of either half) and a second mask make a bf16 pair of them, and one bf16 multiplication with a
// factor for the block gives code * scale (MXFP4) or code * scale * 2^-16 (NVFP4, whose scales reach 448: the
// rest is applied to the sums), exactly. B takes its elements in the same order. The factor of an MXFP4
// scale above 2 (byte > 128) would leave bf16's range and takes a second one; a step that has any, or a NaN scale,
// goes the general way.
static constexpr float kNvfp4Lift = 65536.0f;
template <int W, int MT, int CHUNKS>
struct WeightStep4 {
  static constexpr int kStep = CHUNKS * 128;
  static constexpr int FMT = W == kMoeMxfp4 ? kMxfp4 : kNvfp4;
  static constexpr int kBlocks = 32 / mx_block(FMT);  // block scales of a lane's 32 elements
  uint4 q[MT][2][CHUNKS];
  uint32_t sb[MT][2][CHUNKS];

  template <typename Rows>
  B200_DEVICE void load(const MoeMatrix& w, int k0, int K, uint32_t lane, Rows rows) {
    const uint32_t part = lane & 3u;
    const uint32_t block = static_cast<uint32_t>(k0) / mx_block(FMT) + part * kBlocks;
    const uint8_t* codes = w.data + k0 / 2 + part * 16;
    const uint8_t* scales = w.scales + (block / 4) * kMxGroupBytes + block % 4;
    const long long tile_row = w.col_tiles * mx_tile_bytes(FMT);
#pragma unroll
    for (int m = 0; m < MT; ++m) {
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const int signed_row = rows(m, half);
        const uint32_t row = static_cast<uint32_t>(signed_row);
        const uint8_t* p = codes + row * w.pitch;
        const uint8_t* sp = scales + (row / kMxTileRows) * tile_row + (row % 32) * 16 + (row % kMxTileRows) / 32 * 4;
#pragma unroll
        for (int c = 0; c < CHUNKS; ++c) {
          q[m][half][c] = make_uint4(0u, 0u, 0u, 0u);
          sb[m][half][c] = 0u;
          if (signed_row >= 0 && k0 + c * 128 + static_cast<int>(part) * 32 < K) {
            q[m][half][c] = ptx::ld_stream_v4(p + c * 64);
            if constexpr (FMT == kMxfp4) {
              sb[m][half][c] = sp[c * kMxGroupBytes];
            } else {
              sb[m][half][c] = *reinterpret_cast<const uint16_t*>(sp + c * 2 * kMxGroupBytes);
            }
          }
        }
      }
    }
  }

  // The factor of block `i` of a lane's chunk, in both halves, and the second one.
  template <bool GENERAL>
  B200_DEVICE void factors(uint32_t bytes, int i, uint32_t* first, uint32_t* second) const {
    const uint32_t byte = (bytes >> (8 * i)) & 0xFFu;
    *second = 0x3F803F80u;
    if constexpr (W == kMoeMxfp4) {
      if constexpr (GENERAL) {
        *first = byte == 255u ? 0x7FC07FC0u : min(byte + 126u, 254u) * 0x00800080u;
        if (byte > 128u) *second = (byte - 1u) * 0x00800080u;  // 2^(byte - 128)
      } else {
        *first = byte * 0x00800080u + 126u * 0x00800080u;  // 2^(byte - 1)
      }
    } else {
      // e4m3 bits as a bf16 number are the scale times 2^-120; brought up in two exact steps to 2^110
      const uint32_t bits = byte * 0x00100010u;
      *first = mul_bf16x2(mul_bf16x2(bits, 0x7B807B80u), 0x76807680u);
      if (GENERAL && byte == 0x7Fu) *first = 0x7FC07FC0u;
    }
  }

  // Eight codes as four bf16 pairs (i, i + 4).
  template <bool GENERAL>
  static B200_DEVICE void unpack(uint32_t (&a)[4], uint32_t codes, uint32_t first, uint32_t second) {
    const uint32_t upper = codes >> 8;
    a[0] = ((codes & 0x000F000Fu) * 0x1040u) & 0x81C081C0u;
    a[1] = ((codes & 0x00F000F0u) * 0x0104u) & 0x81C081C0u;
    a[2] = ((upper & 0x000F000Fu) * 0x1040u) & 0x81C081C0u;
    a[3] = ((upper & 0x00F000F0u) * 0x0104u) & 0x81C081C0u;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      a[i] = mul_bf16x2(a[i], first);
      if constexpr (GENERAL && W == kMoeMxfp4) a[i] = mul_bf16x2(a[i], second);
    }
  }

  // NT sums at once, so that a weight is unpacked once: `columns` makes their operands, eight elements as four pairs, of
  // the eight 16-bit words that lie at each of its vectors. GENERAL: any scale, and a step that the end of the
  // rows may cut short.
  template <bool GENERAL, int NT, typename Columns>
  B200_DEVICE void products(float (&acc)[NT][MT][4], const Columns& columns, int k0, int K, uint32_t lane) const {
    const int part = static_cast<int>(lane & 3u);
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c) {
      const int kc = k0 + c * 128 + part * 32;
      uint32_t first[MT][2][kBlocks], second[MT][2][kBlocks];
#pragma unroll
      for (int m = 0; m < MT; ++m) {
#pragma unroll
        for (int half = 0; half < 2; ++half) {
#pragma unroll
          for (int i = 0; i < kBlocks; ++i) factors<GENERAL>(sb[m][half][c], i, &first[m][half][i], &second[m][half][i]);
        }
      }
#pragma unroll
      for (int word = 0; word < 4; ++word) {
        uint4 v[Columns::kReads];
#pragma unroll
        for (int j = 0; j < Columns::kReads; ++j) {
          if constexpr (GENERAL) v[j] = make_uint4(0u, 0u, 0u, 0u);
          if (!GENERAL || kc + word * 8 < K) v[j] = *reinterpret_cast<const uint4*>(columns.at[j] + kc + word * 8);
        }
        uint32_t a[MT][2][4];
        const int i = kBlocks == 2 ? word / 2 : 0;
#pragma unroll
        for (int m = 0; m < MT; ++m) {
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            const uint4& w = q[m][half][c];
            unpack<GENERAL>(a[m][half], word == 0 ? w.x : word == 1 ? w.y : word == 2 ? w.z : w.w, first[m][half][i],
                            second[m][half][i]);
          }
        }
        uint32_t b[NT][4];
        columns.operands(b, v);
#pragma unroll
        for (int j = 0; j < NT; ++j) {
#pragma unroll
          for (int m = 0; m < MT; ++m) {
            mma16816<0>(acc[j][m], a[m][0][0], a[m][1][0], a[m][0][1], a[m][1][1], b[j][0], b[j][1]);
            mma16816<0>(acc[j][m], a[m][0][2], a[m][1][2], a[m][0][3], a[m][1][3], b[j][2], b[j][3]);
          }
        }
      }
    }
  }

  // Column g of tile j is the vector at[j], element after element.
  template <int NT>
  struct Tokens {
    static constexpr int kReads = NT;
    const uint16_t* at[NT];
    B200_DEVICE void operands(uint32_t (&b)[NT][4], const uint4 (&v)[NT]) const {
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        b[j][0] = __byte_perm(v[j].x, v[j].z, 0x5410);
        b[j][1] = __byte_perm(v[j].x, v[j].z, 0x7632);
        b[j][2] = __byte_perm(v[j].y, v[j].w, 0x5410);
        b[j][3] = __byte_perm(v[j].y, v[j].w, 0x7632);
      }
    }
  };
  // Elements i and i + 4 of eight side by side, as unpack() leaves the weights.
  static B200_DEVICE int hidden_place(int i) { return (i & ~7) | (i & 3) << 1 | (i >> 2 & 1); }

  template <int NT, typename Columns>
  B200_DEVICE void mma(float (&acc)[NT][MT][4], const Columns& columns, int k0, int K, uint32_t lane) const {
    if (k0 + kStep > K || general()) {
      products<true>(acc, columns, k0, K, lane);
    } else {
      products<false>(acc, columns, k0, K, lane);
    }
  }
  template <int NT>
  B200_DEVICE void mma_tokens(float (&acc)[NT][MT][4], const uint16_t* const (&b)[NT], int k0, int K, uint32_t lane) const {
    Tokens<NT> columns;
#pragma unroll
    for (int j = 0; j < NT; ++j) columns.at[j] = b[j];
    mma(acc, columns, k0, K, lane);
  }
  template <typename Hidden>
  B200_DEVICE void mma_hidden(float (&acc)[Hidden::kSums][MT][4], const Hidden& columns, int k0, int K, uint32_t lane) const {
    mma(acc, columns, k0, K, lane);
  }

  B200_DEVICE bool general() const {
    bool some = false;
#pragma unroll
    for (int m = 0; m < MT; ++m) {
#pragma unroll
      for (int i = 0; i < 2 * CHUNKS; ++i) {
        const uint32_t bytes = sb[m][i / CHUNKS][i % CHUNKS];
        if constexpr (W == kMoeMxfp4) {
          some = some || bytes > 128u;
        } else {
          some = some || (bytes & 0x7Fu) == 0x7Fu || (bytes & 0x7F00u) == 0x7F00u;
        }
      }
    }
    return __any_sync(0xFFFFFFFFu, some);
  }
};

// MMA tiles of weight rows and steps of the two products: 8 KB on the way per warp, or 4 KB of 4-bit weights, whose rows are a
// quarter as long, so that a unit takes two tiles. 16-bit weights do so in the down product too, with half the step: what
// the parts of the hidden values cost does not grow with the rows (layer of 128 experts (2048, 768), top 8, bf16, against one
// tile: 4 tokens 54.2 against 55.2 us, 16 tokens 123.4 against 125.6, 64 tokens 232 against 235).
template <int W, int F16>
struct MoeUnit {
  using GateUp = WeightStep<F16, 1, 8>;
  using Down = WeightStep<F16, 2, 4>;
  static constexpr int kTiles = 1, kDownTiles = 2;
  static constexpr float kLift = 1.0f;
};
template <>
struct MoeUnit<kMoeMxfp4, 0> {
  using GateUp = WeightStep4<kMoeMxfp4, 2, 2>;
  using Down = WeightStep4<kMoeMxfp4, 2, 2>;
  static constexpr int kTiles = 2, kDownTiles = 2;
  static constexpr float kLift = 1.0f;
};
template <>
struct MoeUnit<kMoeNvfp4, 0> {
  using GateUp = WeightStep4<kMoeNvfp4, 2, 2>;
  using Down = WeightStep4<kMoeNvfp4, 2, 2>;
  static constexpr int kTiles = 2, kDownTiles = 2;
  static constexpr float kLift = kNvfp4Lift;
};

B200_DEVICE float silu(float v) { return __fdiv_rn(v, 1.0f + expf(-v)); }

// The tokens of an expert ride on the MMA's N in the order of its pairs, in the gate/up product two n-tiles at a time (more
// would need more registers than the weights leave). Columns beyond the last token repeat it and are not used.

// ------------------------------------------------------------------------------------- gate and up
// Unit: 8 intermediate columns per MMA tile of one chosen expert = 8 gate rows and the 8 up rows beside them, so that
// a lane ends up with a gate value and its up value. The CTAs take units in turn; a warp issues the next
// step's loads, of the next unit if need be, as soon as its MMAs have taken the registers, so that memory is busy
// while the sums are joined.
struct UnitCursor {
  int index, strip;  // chosen expert, strip of its columns
  B200_DEVICE void advance(int strips, int by_index, int by_strip) {
    index += by_index;
    strip += by_strip;
    if (strip >= strips) {
      strip -= strips;
      ++index;
    }
  }
};

template <int W, int F16>
struct GateUp {
  static constexpr int MT = MoeUnit<W, F16>::kTiles;
  static constexpr int kCols = 8 * MT;
  using Weights = typename MoeUnit<W, F16>::GateUp;
  static constexpr int kStep = Weights::kStep;
  const MoeArgs& args;
  const RouteTables& r;
  uint32_t lane;
  int warp, experts;
  Weights w;

  B200_DEVICE void load(const UnitCursor& u, int k0) {
    const int I = args.I, i0 = u.strip * kCols;
    const int row = r.list[u.index] * 2 * I + i0 + static_cast<int>(lane >> 2);
    w.load(args.w1, k0, args.H, lane, [=](int m, int half) { return m == 0 || i0 + m * 8 < I ? row + m * 8 + (half ? I : 0) : -1; });
  }

  // The loaded step against tiles [j0, j0 + NT) of the unit's tokens; sums go to (first) or on top of `mine`.
  template <int NT>
  B200_DEVICE void tiles(float4* mine, int first_pair, int tokens, int j0, int k0, bool first) {
    const uint16_t* b[NT];
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      const int c = min((j0 + j) * 8 + static_cast<int>(lane >> 2), tokens - 1);
      b[j] = args.x + static_cast<long long>(r.tokens[first_pair + c]) * args.H;
    }
    float acc[NT][MT][4] = {};
    __syncwarp();  // (the MMA wants all lanes together; the sums before it were written under a condition)
    w.mma_tokens(acc, b, k0, args.H, lane);
#pragma unroll
    for (int j = 0; j < NT; ++j) {
#pragma unroll
      for (int m = 0; m < MT; ++m) {
        float4* to = mine + ((j0 + j) * MT + m) * 32 + lane;
        float4 v = make_float4(acc[j][m][0], acc[j][m][1], acc[j][m][2], acc[j][m][3]);
        if (!first) {
          const float4 o = *to;
          v.x += o.x;
          v.y += o.y;
          v.z += o.z;
          v.w += o.w;
        }
        *to = v;
      }
    }
  }

  // `red`: every warp's sums, `stride` float4 apart.
  B200_DEVICE void run(float4* red, int stride, const UnitCursor& unit, const UnitCursor& next) {
    const int tokens = r.size[unit.index], first_pair = r.first[unit.index];
    const int n_tiles = (tokens + 7) / 8;
    const int own = warp * kStep;
    float4* mine = red + warp * stride;
    for (int k0 = own; k0 - own < args.H; k0 += kMoeWarps * kStep) {
      if (k0 < args.H) {
        int j = 0;
        for (; j + 1 < n_tiles; j += 2) tiles<2>(mine, first_pair, tokens, j, k0, k0 == own);
        if (j < n_tiles) tiles<1>(mine, first_pair, tokens, j, k0, k0 == own);
      } else if (k0 == own) {
        for (int i = 0; i < n_tiles * MT; ++i) mine[i * 32 + lane] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      }
      const int k_next = k0 + kMoeWarps * kStep;
      if (k_next - own < args.H) {
        if (k_next < args.H) load(unit, k_next);
      } else if (next.index < experts && own < args.H) {
        load(next, own);
      }
    }
    __syncthreads();
    const int i0 = unit.strip * kCols;
    for (int o = static_cast<int>(threadIdx.x); o < n_tiles * MT * 64; o += kMoeThreads) {
      const int tile = o / 64, row_in = o % 64 / 8, col = o % 8;
      const int c = tile / MT * 8 + col, row = i0 + tile % MT * 8 + row_in;
      if (c >= tokens || row >= args.I) continue;
      const float* at = reinterpret_cast<const float*>(red + tile * 32 + row_in * 4 + col / 2) + (col & 1);
      float gate = at[0], up = at[2];
#pragma unroll
      for (int p = 1; p < kMoeWarps; ++p) {
        gate += at[p * stride * 4];
        up += at[p * stride * 4 + 2];
      }
      const float h = r.weights[first_pair + c] * (silu(gate * args.scale1[0] * args.scale1[1]) * (up * args.scale1[0] * args.scale1[1]));
      uint16_t* to = args.h + static_cast<long long>(r.pairs[first_pair + c]) * 2 * args.I + MoeUnit<W, F16>::Down::hidden_place(row);
      HiddenParts<F16>::store(h, to, to + args.I);
    }
  }
};

__host__ __device__ __forceinline__ int moe_token_tiles(int T) { return (T + 7) / 8; }
// float4 between two warps' sums
__host__ __device__ __forceinline__ int gate_up_stride(int tiles, int T) { return tiles * moe_token_tiles(T) * 32; }
// Sums of two units, used in turn, save a barrier per unit; of one where two CTAs per SM have no room for more (4-bit weights and
// 41 or more tokens: a second buffer left one CTA per SM, the layer 26 us longer for 64 tokens of 128 MXFP4 experts).
__host__ __device__ __forceinline__ int gate_up_buffers(int tiles, int T) {
  return 2 * kMoeWarps * gate_up_stride(tiles, T) * 16 <= 80 * 1024 ? 2 : 1;
}

template <int W, int F16>
__global__ void __launch_bounds__(kMoeThreads, 2) moe_gate_up_kernel(const __grid_constant__ MoeArgs args) {
  constexpr int kCols = GateUp<W, F16>::kCols;
  extern __shared__ __align__(16) uint8_t smem[];
  float4* red = reinterpret_cast<float4*>(smem);
  const int stride = gate_up_stride(MoeUnit<W, F16>::kTiles, args.T);
  const int buffers = gate_up_buffers(MoeUnit<W, F16>::kTiles, args.T);
  const RouteTables r = route_tables_at(smem + buffers * kMoeWarps * stride * 16, args);
  const int strips = (args.I + kCols - 1) / kCols;
  const int by_index = static_cast<int>(gridDim.x) / strips, by_strip = static_cast<int>(gridDim.x) % strips;
  UnitCursor unit{static_cast<int>(blockIdx.x) / strips, static_cast<int>(blockIdx.x) % strips};
  ptx::grid_dependency_wait();
  // Only now: a CTA of the down kernel then starts knowing that the router has completed.
  ptx::grid_launch_dependents();
  build_route_tables(r, args);
  GateUp<W, F16> g{args, r, ptx::lane_id(), static_cast<int>(threadIdx.x) / 32, *r.count, {}};
  if (unit.index < g.experts && g.warp * GateUp<W, F16>::kStep < args.H) g.load(unit, g.warp * GateUp<W, F16>::kStep);
  for (int turn = 0; unit.index < g.experts; turn ^= buffers - 1) {
    UnitCursor next = unit;
    next.advance(strips, by_index, by_strip);
    g.run(red + turn * kMoeWarps * stride, stride, unit, next);
    if (buffers == 1) __syncthreads();
    unit = next;
  }
}

// ------------------------------------------------------------------------------------- down
// Unit: 16 columns of the output per MMA tile, for all tokens, one cluster. The contraction runs over all
// chosen experts; its steps go to the warps of the cluster in turn. An expert's tokens are packed into as few tiles
// as they need; after a step a warp adds its sums to the tokens they belong to, in shared memory of its own
// (a fixed column per token would need no such sums, but an expert's four tokens among 64 then lie in three or four
// tiles of eight: 2.4 times as long for 64 tokens, 128 experts, 2048 x 768).
template <int W, int F16>
struct Down {
  static constexpr int MT = MoeUnit<W, F16>::kDownTiles;
  static constexpr int kPitch = MT * 16 + 1;  // floats between tokens
  using Weights = typename MoeUnit<W, F16>::Down;
  static constexpr int kStep = Weights::kStep;
  const MoeArgs& args;
  const RouteTables& r;
  uint32_t lane;
  int r0, steps;
  Weights w;

  B200_DEVICE void load(int s) {
    const int e = r.list[s / steps];
    const int H = args.H, first = r0 + static_cast<int>(lane >> 2);
    w.load(args.w2, s % steps * kStep, args.I, lane, [=](int m, int half) {
      const int row = first + m * 16 + half * 8;
      return row < H ? e * H + row : -1;
    });
  }

  // The loaded step against the expert's tokens from c0 on, as many as the columns take, on top of the tokens' sums.
  template <typename Hidden>
  B200_DEVICE void tile(float* sums, int first_pair, int tokens, int c0, int k0) {
    constexpr int P = HiddenParts<F16>::kParts, kWidth = 8 / Hidden::kTokens;
    const int column = static_cast<int>(lane >> 2);
    const int token = min(c0 + column / kWidth, tokens - 1);
    const Hidden columns(args.h + static_cast<long long>(r.pairs[first_pair + token]) * 2 * args.I, args.I, column);
    float acc[Hidden::kSums][MT][4] = {};
    __syncwarp();  // (as for the gate/up product)
    w.mma_hidden(acc, columns, k0, args.I, lane);
    // A lane holds columns 2 (lane % 4) and the next one, of rows lane / 4 + 8 m.
    const auto add = [&](int c, auto part) {
      const bool live = c < tokens;
      float* to = sums + r.tokens[first_pair + (live ? c : 0)] * kPitch + (lane >> 2);
#pragma unroll
      for (int m = 0; m < 2 * MT; ++m) {
        float v[P];
#pragma unroll
        for (int p = 0; p < P; ++p) v[p] = part(p, m);
        if (live) to[m * 8] += join_parts<F16>(v);
      }
    };
    const int quad = static_cast<int>(lane & 3u);
    if constexpr (Hidden::kSums == P) {
#pragma unroll
      for (int n = 0; n < 2; ++n) {
        add(c0 + quad * 2 + n, [&](int p, int m) { return acc[p][m / 2][m % 2 * 2 + n]; });
      }
    } else if constexpr (P == 2) {
      add(c0 + quad, [&](int p, int m) { return acc[0][m / 2][m % 2 * 2 + p]; });
    } else {
      // the third part is the next lane's
      add((quad & 1) ? tokens : c0 + quad / 2, [&](int p, int m) {
        return p < 2 ? acc[0][m / 2][m % 2 * 2 + p] : __shfl_xor_sync(0xFFFFFFFFu, acc[0][m / 2][m % 2 * 2], 1);
      });
    }
  }

  B200_DEVICE void run(float* sums, int s, int next, int total) {
    const int tokens = r.size[s / steps], first_pair = r.first[s / steps], k0 = s % steps * kStep;
    using Few = HiddenColumns<F16>;
    using Many = HiddenSums<F16>;
    if (tokens <= Few::kTokens) {
      tile<Few>(sums, first_pair, tokens, 0, k0);
    } else {
      for (int c = 0; c < tokens; c += Many::kTokens) tile<Many>(sums, first_pair, tokens, c, k0);
    }
    if (next < total) load(next);
    __syncwarp();  // the next step's lanes may hold other tokens
  }
};

template <int W, int F16>
__global__ void __launch_bounds__(kMoeThreads, 2) moe_down_kernel(const __grid_constant__ MoeArgs args, int split) {
  using D = Down<W, F16>;
  extern __shared__ __align__(16) uint8_t smem[];
  float* sums = reinterpret_cast<float*>(smem);  // [warp][token][kPitch]
  const int per_warp = args.T * D::kPitch;
  const RouteTables r = route_tables_at(smem + (kMoeWarps * per_warp * 4 + 15) / 16 * 16, args);
  const int warp = static_cast<int>(threadIdx.x) / 32;
  const int rank = split > 1 ? static_cast<int>(ptx::cluster_ctarank()) : 0;
  D d{args, r, ptx::lane_id(), static_cast<int>(blockIdx.x) / split * 16 * D::MT, (args.I + D::kStep - 1) / D::kStep, {}};
  for (int i = static_cast<int>(threadIdx.x); i < kMoeWarps * per_warp; i += kMoeThreads) sums[i] = 0.0f;
  // The routing and the weights are there already: every CTA of the gate/up kernel had waited for the router before this
  // kernel was allowed to start. So the first step's weights are under way while that kernel finishes; its
  // hidden values are what the wait is for.
  build_route_tables(r, args);
  const int total = *r.count * d.steps, stride = split * kMoeWarps;
  int s = rank * kMoeWarps + warp;
  if (s < total) d.load(s);
  ptx::grid_launch_dependents();
  ptx::grid_dependency_wait();
  float* mine = sums + warp * per_warp;
  for (; s < total; s += stride) d.run(mine, s, s + stride, total);
  __syncthreads();
  // The warps' sums into the first warp's, then the CTAs' into the output, in order.
  constexpr int kRows = D::MT * 16;
  for (int i = static_cast<int>(threadIdx.x); i < per_warp; i += kMoeThreads) {
    float v = sums[i];
#pragma unroll
    for (int q = 1; q < kMoeWarps; ++q) v += sums[q * per_warp + i];
    sums[i] = v;
  }
  if (split > 1) {
    ptx::cluster_arrive();
    ptx::cluster_wait();
  } else {
    __syncthreads();
  }
  const uint32_t addr = ptx::smem_u32(sums);
  for (int i = rank * kMoeThreads + static_cast<int>(threadIdx.x); i < args.T * kRows; i += split * kMoeThreads) {
    const int t = i / kRows, row = i % kRows;
    const uint32_t at = static_cast<uint32_t>((t * D::kPitch + row) * 4);
    float v = 0.0f;
#pragma unroll 4
    for (int p = 0; p < split; ++p) v += ptx::ld_cluster_f32(split > 1 ? ptx::map_to_cta(addr + at, p) : addr + at);
    if (d.r0 + row < args.H) args.out[static_cast<long long>(t) * args.H + d.r0 + row] = round16<F16>(v * args.scale2[0] * args.scale2[1]);
  }
  if (split > 1) {
    ptx::cluster_arrive();  // no CTA leaves while another reads its sums
    ptx::cluster_wait();
  }
}

}  // namespace b200
