// Streams of weight fragments for v_mfma_f32_16x16x32, over 4-bit weights with group scales and
// over fp16/bf16 weights: what the 4-bit projections (w4_linear.hip) and the routed experts' layer
// (moe_layer.hip) share.
//
// The product is D[token][weight row] (A = 16 tokens, B = 16 weight rows, 32 k a step): lane l holds
// weight row l % 16 in B and in D, so a row's scale is one value per lane, and D's rows are tokens
// 4 (l / 16) + i.
//
// 4-bit weights. Row n, group g of k: w[n, k] = s[n, g] (q[n, k] - z[n, g]), q and z in 0..15. A code
// becomes the exact value 16 + q with one shift and one and-or for two of them: bits 3..6 (bf16) or
// 6..9 (fp16) of 16.0's mantissa weigh 1..8. The MFMA then sums x (16 + q) exactly as it would any
// fp16/bf16 product, in fp32, and
//   sum x (q - z) = sum x (16 + q) - (16 + z) sum x,
// with sum x over the group from one more MFMA against ones, shared by all rows of the wave. The
// terms are at most 31 / 8 times the size of the products they stand for, so the subtraction costs
// 2 bits of fp32's 24; the scale is applied to the fp32 difference, once per group. No product is
// rounded to 16 bits. An infinite x gives NaN (inf - inf) where the formula's sum would be infinite.
//
// Packed layout: per expert, slabs of 16 rows (gate_up: gate slab 0, up slab 0, gate slab 1, ...),
// each a run of ceil(K / 128) blocks of 1024 + 64 gpb bytes, gpb = 128 / group (1 from 128 on):
//   block[lane][f]: 32-bit word of the codes of row lane % 16 at k = 128 b + 32 f + 8 (lane / 16) + j,
//                   j = 0..7 at bits 4 (j / 2) + 16 (j % 2)          (lane < 64, f < 4)
//   then [row][gpb]: the group's scale as fp32 bits (exact from fp16 or bf16, whose low 13 mantissa
//                   bits are zero) with z in the low four bits.
// One 16-byte load per lane is a whole block's codes, and a slab is one contiguous stream. Groups
// past K and rows past N have scale 0.
#pragma once

#include "ember_common.h"

namespace ember {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

template <typename T>
struct Mfma16;
template <>
struct Mfma16<_Float16> {
  typedef _Float16 v8 __attribute__((ext_vector_type(8)));
  static constexpr uint32_t kOnes = 0x3C003C00u;
  static constexpr uint32_t kMask = 0x03C003C0u, kBias = 0x4C004C00u;  // 16.0, code at mantissa bits 6..9
  static constexpr int kBit = 6;
  static __device__ __forceinline__ f32x4 run(v8 a, v8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
  }
};
template <>
struct Mfma16<__bf16> {
  typedef __bf16 v8 __attribute__((ext_vector_type(8)));
  static constexpr uint32_t kOnes = 0x3F803F80u;
  static constexpr uint32_t kMask = 0x00780078u, kBias = 0x41804180u;  // 16.0, code at mantissa bits 3..6
  static constexpr int kBit = 3;
  static __device__ __forceinline__ f32x4 run(v8 a, v8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
  }
};

// Eight codes of one word as 16 + q.
template <typename T>
__device__ __forceinline__ typename Mfma16<T>::v8 w4_values(uint32_t w) {
  using M = Mfma16<T>;
  u32x4 v;
#pragma unroll
  for (int p = 0; p < 4; ++p) {
    const int sh = M::kBit - 4 * p;
    v[p] = ((sh >= 0 ? w << (sh & 31) : w >> (-sh & 31)) & M::kMask) | M::kBias;
  }
  return __builtin_bit_cast(typename M::v8, v);
}

constexpr int kW4Block = 128;  // k per block

__host__ __device__ inline int w4_gpb(int64_t group) { return group >= kW4Block ? 1 : static_cast<int>(kW4Block / group); }
__host__ __device__ inline int64_t w4_block_bytes(int gpb) { return 1024 + 64 * gpb; }

// A weight matrix as the kernels read it. GPB > 0: 4-bit, groups per block. GPB = 0: fp16/bf16, in
// blocks of 64 k with element strides that cover row-major weights and both packed layouts.
struct WeightView {
  const void* w;
  int64_t es;           // expert stride (4-bit: bytes)
  int64_t s4, s1;       // 16 bits: strides of 64 rows and of 16 rows
  int64_t ps;           // ... of the up half after the gate half
  int64_t bs, hs;       // ... of 64 k and of 32 k
  int64_t lr, lg;       // ... of a row in a fragment and of 8 k
  int parts;            // 4-bit: slabs of one 16-column group (2: gate and up)
  int nb;               // blocks of k
};

// One lane's place in a 16-row slab's stream.
template <typename T, int GPB>
struct WeightPtr {
  const T* p;
  __device__ __forceinline__ void set(const WeightView& v, int64_t e, int slab, int part, int lane) {
    p = static_cast<const T*>(v.w) + e * v.es + (slab >> 2) * v.s4 + (slab & 3) * v.s1 + part * v.ps +
        (lane & 15) * v.lr + (lane >> 4) * v.lg;
  }
};

template <typename T, int R, int NT, int GPB>
struct Stage {
  static constexpr int kFrags = GPB > 0 ? 4 : 2;  // 32-k steps of a block
  static constexpr int kBlock = 32 * kFrags;
  using V8 = typename Mfma16<T>::v8;
  u32x4 w[R][GPB > 0 ? 1 : 2];
  uint32_t m[R][GPB > 0 ? GPB : 1];
  V8 x[NT][kFrags];

  // 4-bit: base = the slab's first byte, uniform. The block's codes and its scales.
  __device__ __forceinline__ void load_w4(int r, const uint8_t* base, int64_t block, int lane) {
    const uint8_t* p = base + block * (1024 + 64 * GPB);
    w[r][0] = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(p + lane * 16));
    const uint8_t* q = p + 1024 + (lane & 15) * (4 * GPB);
    if constexpr (GPB == 4) {
      const u32x4 v = *reinterpret_cast<const u32x4*>(q);
#pragma unroll
      for (int i = 0; i < 4; ++i) m[r][i] = v[i];
    } else if constexpr (GPB == 2) {
      typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
      const u32x2 v = *reinterpret_cast<const u32x2*>(q);
      m[r][0] = v[0];
      m[r][1] = v[1];
    } else {
      m[r][0] = *reinterpret_cast<const uint32_t*>(q);
    }
  }
  // 16 bits: p = this lane's first element of the slab.
  __device__ __forceinline__ void load_half(int r, const T* p, int64_t block, int64_t bs, int64_t hs) {
#pragma unroll
    for (int h = 0; h < 2; ++h)
      w[r][h & (GPB > 0 ? 0 : 1)] = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(p + block * bs + h * hs));
  }
  // The tokens' k of a block: xrow = this lane's token row + 8 (lane / 16). K is a multiple of 32; steps
  // past it re-read the last one (their weights have scale 0).
  __device__ __forceinline__ void load_x(int nt, const T* xrow, int block, int K) {
#pragma unroll
    for (int f = 0; f < kFrags; ++f)
      x[nt][f] = *reinterpret_cast<const V8*>(xrow + min(block * kBlock + 32 * f, K - 32));
  }

  // acc[nt][r] += the block's products.
  __device__ __forceinline__ void compute(f32x4 (&acc)[NT][R]) const {
    using M = Mfma16<T>;
    if constexpr (GPB == 0) {
#pragma unroll
      for (int r = 0; r < R; ++r)
#pragma unroll
        for (int f = 0; f < 2; ++f)
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
            acc[nt][r] = M::run(x[nt][f], __builtin_bit_cast(V8, w[r][f]), acc[nt][r]);
    } else {
      constexpr int FG = 4 / GPB;  // steps of a group within the block
      const V8 ones = __builtin_bit_cast(V8, u32x4{M::kOnes, M::kOnes, M::kOnes, M::kOnes});
      const f32x4 zero = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int g = 0; g < GPB; ++g) {
        f32x4 xs[NT];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          xs[nt] = zero;
#pragma unroll
          for (int f = 0; f < FG; ++f) xs[nt] = M::run(x[nt][g * FG + f], ones, xs[nt]);
        }
#pragma unroll
        for (int r = 0; r < R; ++r) {
          f32x4 part[NT];
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) part[nt] = zero;
#pragma unroll
          for (int f = 0; f < FG; ++f) {
            const V8 wv = w4_values<T>(w[r][0][g * FG + f]);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) part[nt] = M::run(x[nt][g * FG + f], wv, part[nt]);
          }
          const float s = __builtin_bit_cast(float, m[r][g] & ~15u);
          const float z = -16.0f - static_cast<float>(m[r][g] & 15u);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int i = 0; i < 4; ++i)
              acc[nt][r][i] = __builtin_fmaf(s, __builtin_fmaf(z, xs[nt][i], part[nt][i]), acc[nt][r][i]);
        }
      }
    }
  }
};

__device__ __forceinline__ float silu_mul(float g, float u) { return g / (1.0f + expf(-g)) * u; }

}  // namespace ember
