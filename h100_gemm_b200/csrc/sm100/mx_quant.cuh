// Quantisation to microscaled 4-bit floating point and back.
//
// Mathematics, for a block with the largest magnitude a:
//   MXFP4   scale = 2^clamp(floor(log2 a) - 2, -127, 125), from the exponent bits of a
//   NVFP4   scale = s * t, s = RN_e4m3(a / (6 t)) saturating at 448, t the matrix' power of two
//   code    = RN_e2m1(x / scale), ties to even, saturating at 6; s = 0 gives zeros
//   a block that holds a NaN or an infinity gets the NaN scale (and zero codes)
// Everything is exact for 16-bit inputs. Division by 2^e is. For NVFP4, x / t has at most 11
// significant bits and a border between two codes (0.25 or more) times s at most 7, so a quotient x / (s t) that is
// not on a border is 2^-13 away from it or more. x * (1 / (s t)) with a reciprocal good to 2^-22 is within 2^-19 of
// the quotient, and rounded to a multiple of 2^-14 it lies on the border exactly when the quotient does.
// Likewise a / (6 t): rounded to 12 significant bits before it becomes an e4m3 number of four.
//
// Bound by memory: 2 bytes read and 0.53 (MXFP4) or 0.56 (NVFP4) written per element and direction. A CTA
// takes 128 x 128 elements: 256 bytes of every row (whole lines), eight 16-byte loads in flight per
// thread, and complete 512-byte scale groups in either direction, so scales leave as whole lines and
// the padding of the scale layout is written by the CTAs at the edges instead of a memset. The
// transposed form turns the tile in shared memory (34 KB; with 48 to 64 registers per thread four or five CTAs
// per SM); both forms at once read the matrix once.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "mx_format.cuh"
#include "ptx.cuh"

namespace b200 {

static constexpr int kQuantTile = 128;
static constexpr int kQuantThreads = 256;
static constexpr int kQuantPitch = kQuantTile * 2 + 16;  // bytes between rows of the staged tile

struct QuantArgs {
  const uint16_t* x;
  long long rows, cols, ldx;
  float inv_t;              // 1 / tensor scale
  uint8_t* data[2];         // [0] row form, [1] transposed form
  uint8_t* scales[2];
  long long pitch[2];
  long long col_tiles[2];   // scale tiles along a row
  long long row_tiles[2];
  int tiles_x;              // CTAs along the columns of x
};

template <int F16>
__device__ __forceinline__ float half_bits_to_float(uint32_t bits) {
  if constexpr (F16) {
    return __half2float(__ushort_as_half(static_cast<unsigned short>(bits)));
  } else {
    return __uint_as_float(bits << 16);
  }
}

// Elements [lo, hi) of the eight at src, the others zero.
__device__ __forceinline__ void load_elements(uint32_t (&w)[4], const uint16_t* src, int lo, int hi) {
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    if (j >= lo && j < hi) w[j / 2] |= static_cast<uint32_t>(src[j]) << (16 * (j & 1));
  }
}

// Eight 16-bit elements from element `at` of a row in shared memory (the row itself starts on 4 bytes).
__device__ __forceinline__ void read_shifted(uint32_t (&w)[4], const uint8_t* row, int at) {
  const uint32_t* words = reinterpret_cast<const uint32_t*>(row) + (at >> 1);
  uint32_t v[5];
#pragma unroll
  for (int k = 0; k < 5; ++k) v[k] = (k < 4 || (at & 1)) ? words[k] : 0u;
#pragma unroll
  for (int k = 0; k < 4; ++k) w[k] = (at & 1) ? __funnelshift_r(v[k], v[k + 1], 16) : v[k];
}

// The scale byte of a block whose largest magnitude is `amax` (as bits), and its factor: what the elements are
// multiplied with; negative where they are first to be clipped to 2688 t (their product would leave
// fp32's range), NaN for a block that holds a NaN or an infinity.
template <int FMT, int F16>
__device__ __forceinline__ float block_scale(uint32_t amax, float inv_t, uint32_t* byte) {
  const bool bad = amax >= (F16 ? 0x7C00u : 0x7F80u);
  const float a = half_bits_to_float<F16>(amax);
  float factor;
  if constexpr (FMT == kMxfp4) {
    const int e = static_cast<int>(__float_as_uint(a) >> 23) - 2;  // biased exponent of the scale
    const uint32_t b = static_cast<uint32_t>(e > 0 ? e : 0);
    *byte = bad ? 255u : b;
    factor = __uint_as_float((254u - b) << 23);
  } else {
    const float scaled = a * inv_t;
    const float sixth = fminf(scaled, 2688.0f) * (1.0f / 6.0f);
    const float c = sixth * 4097.0f;
    const uint32_t b = e4m3_byte(__fsub_rn(c, __fsub_rn(c, sixth)));
    *byte = bad ? 127u : b;
    float r;
    asm("rcp.approx.f32 %0, %1;" : "=f"(r) : "f"(__uint_as_float(b << 20) * 1.329227995784916e36f));  // (e4m3_value)
    factor = b == 0u ? 0.0f : scaled > 2688.0f ? -r : r * inv_t;
  }
  return bad ? __uint_as_float(0x7FC00000u) : factor;
}

// Two fp32 numbers at once: the SM's packed arithmetic halves what an element costs.
struct Pair {
  uint64_t v;
};
__device__ __forceinline__ Pair pair_of(float lo, float hi) {
  Pair p;
  asm("mov.b64 %0, {%1, %2};" : "=l"(p.v) : "f"(lo), "f"(hi));
  return p;
}
__device__ __forceinline__ Pair pair_mul(Pair a, Pair b) {
  Pair p;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(p.v) : "l"(a.v), "l"(b.v));
  return p;
}
__device__ __forceinline__ Pair pair_fma(Pair a, Pair b, Pair c) {
  Pair p;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(p.v) : "l"(a.v), "l"(b.v), "l"(c.v));
  return p;
}
__device__ __forceinline__ Pair pair_add(Pair a, Pair b) {
  Pair p;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(p.v) : "l"(a.v), "l"(b.v));
  return p;
}

// The larger of the magnitudes of two pairs of 16-bit numbers (NaN wins), with signs to be ignored.
template <int F16>
__device__ __forceinline__ uint32_t max_magnitude2(uint32_t a, uint32_t b) {
  uint32_t r;
  if constexpr (F16) {
    asm("max.NaN.xorsign.abs.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  } else {
    asm("max.NaN.xorsign.abs.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  }
  return r;
}

// Eight elements (two to a word) -> eight codes.
template <int FMT, int F16>
__device__ __forceinline__ uint32_t quantise8(const uint32_t (&w)[4], float inv_t, float factor) {
  float v[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    v[j] = half_bits_to_float<F16>((j & 1) ? w[j / 2] >> 16 : w[j / 2] & 0xFFFFu);
  }
  if constexpr (FMT == kNvfp4) {
    if (factor < 0.0f) {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = fminf(fmaxf(v[j] * inv_t, -2688.0f), 2688.0f);
    }
  }
  const float m = FMT == kNvfp4 ? fabsf(factor) : factor;
  const Pair mm = pair_of(m, m);
#pragma unroll
  for (int j = 0; j < 8; j += 2) {
    Pair p = pair_of(v[j], v[j + 1]);
    if constexpr (FMT == kNvfp4) {
      constexpr float kRound = 768.0f;  // numbers from 512 to 1024 are multiples of 2^-14
      p = pair_add(pair_fma(p, mm, pair_of(kRound, kRound)), pair_of(-kRound, -kRound));
    } else {
      p = pair_mul(p, mm);
    }
    asm("mov.b64 {%0, %1}, %2;" : "=f"(v[j]), "=f"(v[j + 1]) : "l"(p.v));
  }
  const uint32_t codes = e2m1_pack8(v);
  return factor == factor ? codes : 0u;
}

// ROW / COL: which forms are written. VEC: rows of x start on 16 bytes.
template <int FMT, int F16, int ROW, int COL, int VEC>
__global__ void __launch_bounds__(kQuantThreads) quantize_kernel(const __grid_constant__ QuantArgs args) {
  constexpr int kGroups = kQuantTile / (4 * mx_block(FMT));  // scale groups of this tile: 1 or 2
  __shared__ __align__(16) uint8_t tile[COL || !VEC ? kQuantTile * kQuantPitch : 16];
  __shared__ __align__(16) uint8_t scale_row[ROW ? kGroups * kMxGroupBytes : 16];
  __shared__ __align__(16) uint8_t scale_col[COL ? kGroups * kMxGroupBytes : 16];
  const int t = static_cast<int>(threadIdx.x);
  const long long tx = blockIdx.x % args.tiles_x, ty = blockIdx.x / args.tiles_x;
  const long long r0 = ty * kQuantTile, c0 = tx * kQuantTile;
  const int piece = t & 15;  // 8 columns
  const long long col = c0 + piece * 8;
  ptx::grid_launch_dependents();
  ptx::grid_dependency_wait();

  uint32_t w[8][4];
  if constexpr (VEC) {
#pragma unroll
    for (int p = 0; p < 8; ++p) {
      const long long row = r0 + p * 16 + (t >> 4);
      w[p][0] = w[p][1] = w[p][2] = w[p][3] = 0u;
      if (row < args.rows) {
        const uint16_t* src = args.x + row * args.ldx + col;
        if (col + 8 <= args.cols) {
          const uint4 q = ptx::ld_stream_v4(src);
          w[p][0] = q.x;
          w[p][1] = q.y;
          w[p][2] = q.z;
          w[p][3] = q.w;
        } else {
          load_elements(w[p], src, 0, static_cast<int>(args.cols - col));
        }
      }
    }
  } else {
    // Rows off 16 bytes: the aligned pieces that cover a row of the tile go to shared memory as they lie, and
    // every thread takes its eight elements from there (element by element the loads took three times as long).
    uint4 piece_data[9];
    const int lane16 = t & 15;
#pragma unroll
    for (int p = 0; p < 9; ++p) {
      // (eight passes of 16 pieces, then the seventeenth pieces of all rows)
      const int r = p < 8 ? p * 16 + (t >> 4) : t;
      const int k = p < 8 ? lane16 : 16;
      const long long row = r0 + r;
      uint32_t e[4] = {0u, 0u, 0u, 0u};
      if (r < kQuantTile && row < args.rows) {
        const uint16_t* src = args.x + row * args.ldx + c0;
        const int from = k * 8 - static_cast<int>(reinterpret_cast<uintptr_t>(src) & 15u) / 2;  // of the tile's columns
        if (c0 + from >= 0 && c0 + from + 8 <= args.cols) {
          const uint4 q = ptx::ld_stream_v4(src + from);
          e[0] = q.x;
          e[1] = q.y;
          e[2] = q.z;
          e[3] = q.w;
        } else {
          const long long lo = -(c0 + from), hi = args.cols - (c0 + from);
          load_elements(e, src + from, lo > 0 ? static_cast<int>(lo) : 0, hi < 8 ? static_cast<int>(hi) : 8);
        }
      }
      piece_data[p] = make_uint4(e[0], e[1], e[2], e[3]);
    }
#pragma unroll
    for (int p = 0; p < 9; ++p) {
      const int r = p < 8 ? p * 16 + (t >> 4) : t;
      if (r < kQuantTile) *reinterpret_cast<uint4*>(tile + r * kQuantPitch + (p < 8 ? lane16 : 16) * 16) = piece_data[p];
    }
    __syncthreads();
#pragma unroll
    for (int p = 0; p < 8; ++p) {
      const int r = p * 16 + (t >> 4);
      const int lead = static_cast<int>(reinterpret_cast<uintptr_t>(args.x + (r0 + r) * args.ldx + c0) & 15u) / 2;
      read_shifted(w[p], tile + r * kQuantPitch, piece * 8 + lead);
    }
    if constexpr (COL) __syncthreads();  // (the tile takes the same elements again, in place)
  }

  if constexpr (COL) {
#pragma unroll
    for (int p = 0; p < 8; ++p) {
      *reinterpret_cast<uint4*>(tile + (p * 16 + (t >> 4)) * kQuantPitch + piece * 16) =
          make_uint4(w[p][0], w[p][1], w[p][2], w[p][3]);
    }
  }
  if constexpr (ROW) {
    constexpr int kLanes = mx_block(FMT) / 8;  // lanes that share a block
    // Two passes at a time: the lanes of an NVFP4 block each work out the scale of one of them (the scale costs as
    // much as eight elements) and exchange the factors.
#pragma unroll
    for (int p = 0; p < 8; p += 2) {
      uint32_t m[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint32_t(&v)[4] = w[p + h];
        m[h] = max_magnitude2<F16>(max_magnitude2<F16>(v[0], v[1]), max_magnitude2<F16>(v[2], v[3]));
        m[h] = max(m[h] & 0x7FFFu, (m[h] >> 16) & 0x7FFFu);
        m[h] = max(m[h], __shfl_xor_sync(0xFFFFFFFFu, m[h], 1));
        if constexpr (FMT == kMxfp4) m[h] = max(m[h], __shfl_xor_sync(0xFFFFFFFFu, m[h], 2));
      }
      float factor[2];
      uint32_t byte;
      const int own = piece & 1;  // the pass whose scale this lane works out
      const float mine = block_scale<FMT, F16>(own ? m[1] : m[0], args.inv_t, &byte);
      const float other = __shfl_xor_sync(0xFFFFFFFFu, mine, 1);
      factor[0] = own ? other : mine;
      factor[1] = own ? mine : other;
      if (piece % kLanes < 2) {
        const int block = piece / kLanes, r = (p + own) * 16 + (t >> 4);
        scale_row[(block / 4) * kMxGroupBytes + (r % 32) * 16 + (r / 32) * 4 + block % 4] = static_cast<uint8_t>(byte);
      }
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint32_t codes = quantise8<FMT, F16>(w[p + h], args.inv_t, factor[h]);
        const long long row = r0 + (p + h) * 16 + (t >> 4);
        if (row < args.rows && col / 2 + 4 <= args.pitch[0]) {
          *reinterpret_cast<uint32_t*>(args.data[0] + row * args.pitch[0] + col / 2) = codes;
        }
      }
    }
  }
  __syncthreads();
  if constexpr (ROW) {
    // (with both forms the grid covers the padding of either; tiles outside this form's own are not written)
    if (t < kGroups * kMxGroupBytes / 16 && ty < args.row_tiles[0] && tx < 2 * args.col_tiles[0]) {
      uint8_t* dst = args.scales[0] + (ty * args.col_tiles[0] * 2 + tx) * (kGroups * kMxGroupBytes);
      reinterpret_cast<uint4*>(dst)[t] = reinterpret_cast<const uint4*>(scale_row)[t];
    }
  }
  if constexpr (COL) {
    // Thread: columns 2 cp and 2 cp + 1, 32 consecutive rows of x (= elements of the transposed row).
    const int cp = t & 63, rb = t >> 6;
    uint32_t codes[2][4];
    uint32_t v[32];
#pragma unroll
    for (int j = 0; j < 32; ++j) {
      v[j] = *reinterpret_cast<const uint32_t*>(tile + (rb * 32 + j) * kQuantPitch + cp * 4);
    }
    constexpr int kBlk = mx_block(FMT);
#pragma unroll
    for (int b = 0; b < 32 / kBlk; ++b) {
      uint32_t m = v[b * kBlk];
#pragma unroll
      for (int j = 1; j < kBlk; ++j) m = max_magnitude2<F16>(m, v[b * kBlk + j]);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        uint32_t byte;
        const float factor = block_scale<FMT, F16>((h ? m >> 16 : m) & 0x7FFFu, args.inv_t, &byte);
#pragma unroll
        for (int g = 0; g < kBlk / 8; ++g) {
          const uint32_t* s = &v[b * kBlk + g * 8];
          const uint32_t sel = h ? 0x7632u : 0x5410u;  // the upper or lower halves of two words
          const uint32_t e[4] = {__byte_perm(s[0], s[1], sel), __byte_perm(s[2], s[3], sel),
                                 __byte_perm(s[4], s[5], sel), __byte_perm(s[6], s[7], sel)};
          codes[h][b * (kBlk / 8) + g] = quantise8<FMT, F16>(e, args.inv_t, factor);
        }
        const int r = cp * 2 + h, block = rb * (32 / kBlk) + b;
        scale_col[(block / 4) * kMxGroupBytes + (r % 32) * 16 + (r / 32) * 4 + block % 4] = static_cast<uint8_t>(byte);
      }
    }
    __syncthreads();  // the tile has been read: it now takes the codes, 64 bytes per transposed row
    constexpr int kOutPitch = 80;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      *reinterpret_cast<uint4*>(tile + (cp * 2 + h) * kOutPitch + rb * 16) =
          make_uint4(codes[h][0], codes[h][1], codes[h][2], codes[h][3]);
    }
    __syncthreads();
#pragma unroll
    for (int i = t; i < kQuantTile * 4; i += kQuantThreads) {
      const long long row = c0 + i / 4, at = r0 / 2 + (i % 4) * 16;
      if (row < args.cols && at + 16 <= args.pitch[1]) {
        *reinterpret_cast<uint4*>(args.data[1] + row * args.pitch[1] + at) =
            *reinterpret_cast<const uint4*>(tile + (i / 4) * kOutPitch + (i % 4) * 16);
      }
    }
    if (t < kGroups * kMxGroupBytes / 16 && tx < args.row_tiles[1] && ty < 2 * args.col_tiles[1]) {
      uint8_t* dst = args.scales[1] + (tx * args.col_tiles[1] * 2 + ty) * (kGroups * kMxGroupBytes);
      reinterpret_cast<uint4*>(dst)[t] = reinterpret_cast<const uint4*>(scale_col)[t];
    }
  }
}

struct DequantArgs {
  const uint8_t* data;
  const uint8_t* scales;
  long long rows, cols, pitch, col_tiles;
  float tensor_scale;
  int inexact;              // 1: the tensor scale is no power of two
  uint16_t* x;
  long long ldx;
  int tiles_x;
};

// v * t, where fp32 has to round it, rounded to odd: the last bit says that something was cut off, so the rounding to 16 bits
// that follows is the only one. (Below fp32's normal numbers what was cut off may be lost.)
__device__ __forceinline__ float product_to_odd(float v, float t) {
  const float p = __fmul_rn(v, t);
  const float rest = fmaf(v, t, -p);
  if (rest == 0.0f) return p;
  const uint32_t bits = __float_as_uint(p) - ((rest < 0.0f) != (p < 0.0f) ? 1u : 0u);  // towards zero
  return __uint_as_float(bits | 1u);
}

template <int FMT, int F16>
__device__ __forceinline__ void dequantise8(uint32_t (&w)[4], uint32_t codes, float scale, float tensor_scale, int inexact) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    float lo = e2m1_value(codes >> (8 * j)) * scale;
    float hi = e2m1_value(codes >> (8 * j + 4)) * scale;
    if constexpr (FMT == kNvfp4) {
      lo = inexact ? product_to_odd(lo, tensor_scale) : lo * tensor_scale;
      hi = inexact ? product_to_odd(hi, tensor_scale) : hi * tensor_scale;
    }
    if constexpr (F16) {
      asm("cvt.rn.f16x2.f32 %0, %2, %1;" : "=r"(w[j]) : "f"(lo), "f"(hi));
    } else {
      asm("cvt.rn.bf16x2.f32 %0, %2, %1;" : "=r"(w[j]) : "f"(lo), "f"(hi));
    }
  }
}

// Codes and scales -> 16-bit values: code * scale * tensor scale in fp32, rounded once (under a tensor scale that is a power
// of two exact in bf16 unless it leaves bf16's range: 2 bits of code times at most 4 of scale). Same 128 x 128 tiles.
template <int FMT, int F16, int VEC>
__global__ void __launch_bounds__(kQuantThreads) dequantize_kernel(const __grid_constant__ DequantArgs args) {
  const int t = static_cast<int>(threadIdx.x);
  const long long tx = blockIdx.x % args.tiles_x, ty = blockIdx.x / args.tiles_x;
  const long long col = tx * kQuantTile + (t & 15) * 8;
  __shared__ __align__(16) uint8_t tile[VEC ? 16 : kQuantTile * kQuantPitch];
  ptx::grid_launch_dependents();
  ptx::grid_dependency_wait();
  uint32_t codes[8];
#pragma unroll
  for (int p = 0; p < 8; ++p) {
    const long long row = ty * kQuantTile + p * 16 + (t >> 4);
    codes[p] = 0u;
    if (row < args.rows && col < args.cols) {
      codes[p] = *reinterpret_cast<const uint32_t*>(args.data + row * args.pitch + col / 2);
    }
  }
  // The scales of four of a thread's rows lie in 16 bytes of a group: those of its even and those of its odd
  // passes. (The layout is padded to whole tiles.)
  const long long block = (col < args.cols ? col : 0) / mx_block(FMT);
  const uint8_t* group = args.scales + mx_scale_offset(FMT, ty * kQuantTile, block / 4 * 4, args.col_tiles);
  uint32_t scales[2][4];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const uint4 q = *reinterpret_cast<const uint4*>(group + (h * 16 + (t >> 4)) * 16);
    scales[h][0] = q.x;
    scales[h][1] = q.y;
    scales[h][2] = q.z;
    scales[h][3] = q.w;
  }
#pragma unroll
  for (int p = 0; p < 8; ++p) {
    const long long row = ty * kQuantTile + p * 16 + (t >> 4);
    if (row >= args.rows || col >= args.cols) continue;
    const float scale = mx_scale_value<FMT>((scales[p & 1][p / 2] >> (8 * static_cast<int>(block % 4))) & 0xFFu);
    uint32_t w[4];
    dequantise8<FMT, F16>(w, codes[p], scale, args.tensor_scale, args.inexact);
    if constexpr (VEC) {
      uint16_t* dst = args.x + row * args.ldx + col;
      if (col + 8 <= args.cols) {
        *reinterpret_cast<uint4*>(dst) = make_uint4(w[0], w[1], w[2], w[3]);
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          if (col + j < args.cols) dst[j] = static_cast<uint16_t>(w[j / 2] >> (16 * (j & 1)));
        }
      }
    } else {
      *reinterpret_cast<uint4*>(tile + (p * 16 + (t >> 4)) * kQuantPitch + (t & 15) * 16) = make_uint4(w[0], w[1], w[2], w[3]);
    }
  }
  if constexpr (!VEC) {
    // Rows off 16 bytes: every aligned piece of x that starts in this tile is written whole, by 16 threads per row; the
    // values it needs of the next tile's first eight columns are worked out here as well. (Element by element,
    // 4999 x 5005 took 79 us; with pieces cut at the tiles' edges 24 us.)
    const long long c0 = tx * kQuantTile;
    if (t < kQuantTile) {
      const long long row = ty * kQuantTile + t, next = c0 + kQuantTile;
      if (row < args.rows && next < args.cols) {
        const uint32_t word = *reinterpret_cast<const uint32_t*>(args.data + row * args.pitch + next / 2);
        const uint32_t byte = args.scales[mx_scale_offset(FMT, row, next / mx_block(FMT), args.col_tiles)];
        uint32_t w[4];
        dequantise8<FMT, F16>(w, word, mx_scale_value<FMT>(byte), args.tensor_scale, args.inexact);
        *reinterpret_cast<uint4*>(tile + t * kQuantPitch + kQuantTile * 2) = make_uint4(w[0], w[1], w[2], w[3]);
      }
    }
    __syncthreads();
#pragma unroll 4
    for (int p = 0; p < 8; ++p) {
      const int r = p * 16 + (t >> 4);
      const long long row = ty * kQuantTile + r;
      if (row >= args.rows) break;
      uint16_t* dst = args.x + row * args.ldx + c0;
      const int head = static_cast<int>((16u - (reinterpret_cast<uintptr_t>(dst) & 15u)) & 15u) / 2;
      const int e = head + (t & 15) * 8;
      const int left = static_cast<int>(args.cols - c0 < 2 * kQuantTile ? args.cols - c0 : 2 * kQuantTile) - e;
      const uint16_t* src = reinterpret_cast<const uint16_t*>(tile + r * kQuantPitch);
      if (left >= 8) {
        uint32_t v[4];
        read_shifted(v, tile + r * kQuantPitch, e);
        *reinterpret_cast<uint4*>(dst + e) = make_uint4(v[0], v[1], v[2], v[3]);
      } else {
        for (int k = 0; k < left; ++k) dst[e + k] = src[e + k];  // the row's end
      }
      if (c0 == 0 && (t & 15) == 0) {
        const int first = head < args.cols ? head : static_cast<int>(args.cols);
        for (int k = 0; k < first; ++k) dst[k] = src[k];  // its beginning
      }
    }
  }
}

}  // namespace b200
