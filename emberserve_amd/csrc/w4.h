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
// rounded to 16 bits. An infinite x, or one so large that a
// group's sum of 31 x overflows fp32 (bf16, 2^116 and more), gives NaN (inf - inf) or an infinity.
//
// Packed layout: per expert, slabs of 16 rows (gate_up: gate slab 0, up slab 0, gate slab 1, ...). A slab
// is nb = ceil(K / 128) blocks of 1 KiB of codes, then the scales of all blocks, rounded up to 128 bytes:
//   block[lane][f]: 32-bit word of the codes of row lane % 16 at k = 128 b + 32 f + 8 (lane / 16) + j,
//                   j = 0..7 at bits 4 (j / 2) + 16 (j % 2)          (lane < 64, f < 4)
//   scales[block][row][gpb]: gpb = 128 / group groups a block (1 from 128 on), each the scale as fp32 bits
//                   (exact from fp16 or bf16, whose low 13 mantissa bits are zero) with z in the low four.
// One 16-byte load per lane is a whole block's codes, and a block is whole 128-byte lines: with the scales
// right behind each block, the lines that two blocks shared came from memory twice (7% more traffic at
// groups of 128). Groups past K and rows past N have scale 0.
#pragma once

#include "ember_common.h"

namespace ember {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

typedef __amdgpu_buffer_rsrc_t BufferRsrc;
constexpr int kPolicyNt = 2;  // non-temporal

// An offset to OR into a load's: past every resource (the load gives zeros) where `past`, else 0. Opaque,
// or the compiler turns the choice into a branch around every load.
__device__ __forceinline__ int nowhere(bool past) {
  int v = past ? 0x7fffff00 : 0;
#if defined(__HIP_DEVICE_COMPILE__)
  asm("" : "+v"(v));
#endif
  return v;
}

__device__ __forceinline__ BufferRsrc buffer(const void* base, int bytes) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(base), 0, bytes, kBufferWord3);
}

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

// (w & mask) | bias as one v_and_or_b32: gfx9 takes one scalar and no literal in it, so the mask has to sit
// in a vector register, which the empty asm makes the compiler do; it splits two literals into two
// instructions (12 a word of codes instead of 8).
__device__ __forceinline__ uint32_t and_or(uint32_t w, uint32_t mask, uint32_t bias) {
#if defined(__HIP_DEVICE_COMPILE__)
  asm("" : "+v"(mask));
#endif
  return (w & mask) | bias;
}

// Eight codes of one word as 16 + q.
template <typename T>
__device__ __forceinline__ typename Mfma16<T>::v8 w4_values(uint32_t w) {
  using M = Mfma16<T>;
  u32x4 v;
#pragma unroll
  for (int p = 0; p < 4; ++p) {
    const int sh = M::kBit - 4 * p;
    v[p] = and_or(sh >= 0 ? w << (sh & 31) : w >> (-sh & 31), M::kMask, M::kBias);
  }
  return __builtin_bit_cast(typename M::v8, v);
}

constexpr int kW4Block = 128;  // k per block

__host__ __device__ inline int w4_gpb(int64_t group) { return group >= kW4Block ? 1 : static_cast<int>(kW4Block / group); }
__host__ __device__ inline int64_t w4_slab_bytes(int64_t nb, int gpb) { return nb * 1024 + (nb * 64 * gpb + 127) / 128 * 128; }

// A workgroup barrier that waits for this wave's LDS accesses but not for its global loads (__syncthreads()
// would drain the loads in flight). The asm keeps memory accesses from moving across it.
__device__ __forceinline__ void lds_barrier() {
  __builtin_amdgcn_s_waitcnt(15 | (3 << 14) | (7 << 4));  // lgkmcnt(0)
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// One block of R slabs, as loaded.
template <int R, int GPB>
struct W4Block {
  u32x4 w[R];
  uint32_t m[R][GPB];

  // slab: the slab's bytes. Buffer loads: the address is the resource, a scalar and one lane offset, so
  // that no vector arithmetic goes into it.
  __device__ __forceinline__ void load(int r, BufferRsrc slab, int block, int nb, int lane) {
    w[r] = __builtin_amdgcn_raw_buffer_load_b128(slab, lane * 16, block * 1024, kPolicyNt);
    const int at = nb * 1024 + block * (64 * GPB);
    const int mo = (lane & 15) * (4 * GPB);
    if constexpr (GPB == 4) {
      const u32x4 v = __builtin_amdgcn_raw_buffer_load_b128(slab, mo, at, 0);
#pragma unroll
      for (int i = 0; i < 4; ++i) m[r][i] = v[i];
    } else if constexpr (GPB == 2) {
      const u32x2 v = __builtin_amdgcn_raw_buffer_load_b64(slab, mo, at, 0);
      m[r][0] = v[0];
      m[r][1] = v[1];
    } else {
      m[r][0] = __builtin_amdgcn_raw_buffer_load_b32(slab, mo, at, 0);
    }
  }

  // acc[nt][r] += the block's products with the fragments x(nt, f).
  template <typename T, int NT, typename X>
  __device__ __forceinline__ void compute(X x, f32x4 (&acc)[NT][R]) const {
    using M = Mfma16<T>;
    using V8 = typename M::v8;
    constexpr int FG = 4 / GPB;  // 32-k steps of a group
    const V8 ones = __builtin_bit_cast(V8, u32x4{M::kOnes, M::kOnes, M::kOnes, M::kOnes});
    const f32x4 zero = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int g = 0; g < GPB; ++g) {
      f32x4 xs[NT], part[NT][R];
      auto scale = [&](int r) {
        const float s = __builtin_bit_cast(float, m[r][g] & ~15u);
        const float z = -16.0f - static_cast<float>(m[r][g] & 15u);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
          for (int i = 0; i < 4; ++i)
            acc[nt][r][i] = __builtin_fmaf(s, __builtin_fmaf(z, xs[nt][i], part[nt][r][i]), acc[nt][r][i]);
#if defined(__HIP_DEVICE_COMPILE__)
          // the sums are made here: put off, the parts of every group and slab are live at once, and spill
          asm volatile("" : "+v"(acc[nt][r]));
#endif
        }
      };
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        xs[nt] = zero;
#pragma unroll
        for (int r = 0; r < R; ++r) part[nt][r] = zero;
      }
      if constexpr (R > 2) {  // slab by slab: fewer registers
        V8 xv[NT][FG];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int f = 0; f < FG; ++f) {
            xv[nt][f] = __builtin_bit_cast(V8, x(nt, g * FG + f));
            xs[nt] = M::run(xv[nt][f], ones, xs[nt]);
          }
#pragma unroll
        for (int r = 0; r < R; ++r) {
#pragma unroll
          for (int f = 0; f < FG; ++f) {
            const V8 wv = w4_values<T>(w[r][g * FG + f]);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) part[nt][r] = M::run(xv[nt][f], wv, part[nt][r]);
          }
          scale(r);
        }
      } else {  // step by step: the chains of all slabs and tiles side by side (3% faster at one token)
#pragma unroll
        for (int f = 0; f < FG; ++f) {
          V8 xv[NT], wv[R];
#pragma unroll
          for (int r = 0; r < R; ++r) wv[r] = w4_values<T>(w[r][g * FG + f]);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            xv[nt] = __builtin_bit_cast(V8, x(nt, g * FG + f));
            xs[nt] = M::run(xv[nt], ones, xs[nt]);
#pragma unroll
            for (int r = 0; r < R; ++r) part[nt][r] = M::run(xv[nt], wv[r], part[nt][r]);
          }
        }
#pragma unroll
        for (int r = 0; r < R; ++r) scale(r);
      }
    }
  }
};

// A wave's tokens of one block: NT tiles of 4 XI rows. A load takes 4 rows' whole 256 bytes (a fragment's
// own order would touch 64 lines an instruction: 2 us more at 16 tokens); the wave's piece of LDS turns
// them into fragments. Row r's 16-byte piece p sits at p ^ r, so that neither side meets a bank twice.
template <int NT, int XI>
struct XBlock {
  static constexpr int kPieces = 64 * XI * NT;  // of the wave's LDS
  u32x4 x[NT * XI];

  // off[i]: this lane's byte offset of row 4 i + lane / 16 and piece lane % 16 of block 0.
  __device__ __forceinline__ void load(BufferRsrc rows, const int (&off)[NT * XI], int block, int k, int lane) {
    const int past = nowhere(block * kW4Block + 8 * (lane & 15) >= k);
#pragma unroll
    for (int i = 0; i < NT * XI; ++i)
      x[i] = __builtin_amdgcn_raw_buffer_load_b128(rows, off[i] | past, block * (2 * kW4Block), 0);
  }
  __device__ __forceinline__ void put(u32x4* lds, int lane) const {
    asm volatile("" ::: "memory");  // the reads of the block before are over: LDS answers a wave in order
#pragma unroll
    for (int i = 0; i < NT * XI; ++i) {
      const int r = 4 * i + (lane >> 4);
      lds[16 * r + ((lane & 15) ^ (r & 15))] = x[i];
    }
    asm volatile("" ::: "memory");
  }
  static __device__ __forceinline__ u32x4 frag(const u32x4* lds, int nt, int f, int lane) {
    const int r = lane & (4 * XI - 1);
    return lds[16 * (16 * nt + r) + ((4 * f + (lane >> 4)) ^ r)];
  }
};

// A wave's stream of items [first, end), D of them in flight.
template <typename S, int D, typename Issue, typename Consume>
__device__ __forceinline__ void stream(int first, int end, Issue issue, Consume consume) {
  if (first >= end) return;
  S ring[D];
#pragma unroll
  for (int d = 0; d < D; ++d) {
    issue(ring[d], first + d);
    __builtin_amdgcn_sched_barrier(0);  // in the ring's order, the oldest consumed first
  }
  int j = first;
  for (; j + D < end; j += D) {
#pragma unroll
    for (int d = 0; d < D; ++d) {
      consume(ring[d], j + d);
      issue(ring[d], j + D + d);
      __builtin_amdgcn_sched_barrier(0);
    }
  }
#pragma unroll
  for (int d = 0; d < D; ++d)
    if (j + d < end) consume(ring[d], j + d);
}

// A 16-bit weight matrix of experts, in blocks of 64 k, by element strides that cover row-major weights
// and both packed layouts; or a packed 4-bit one (w, es in bytes, nb).
struct WeightView {
  const void* w;
  int64_t es;       // expert stride
  int64_t s4, s1;   // 64 rows and 16 rows
  int64_t ps;       // the up half after the gate half
  int64_t bs, hs;   // 64 k and 32 k
  int64_t lr, lg;   // a row in a fragment and 8 k
  int nb;           // blocks of k
};

template <typename T>
__device__ __forceinline__ const T* half_slab(const WeightView& v, int64_t e, int slab, int part, int lane) {
  return static_cast<const T*>(v.w) + e * v.es + (slab >> 2) * v.s4 + (slab & 3) * v.s1 + part * v.ps +
         (lane & 15) * v.lr + (lane >> 4) * v.lg;
}

// A block of R slabs of 16-bit weights and its 16 tokens, in fragment order.
template <typename T, int R>
struct HalfStage {
  using V8 = typename Mfma16<T>::v8;
  u32x4 w[R][2];
  V8 x[2];

  __device__ __forceinline__ void load(int r, const T* p, int64_t block, int64_t bs, int64_t hs) {
#pragma unroll
    for (int h = 0; h < 2; ++h)
      w[r][h] = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(p + block * bs + h * hs));
  }
  __device__ __forceinline__ void load_x(const T* xrow, int block) {
#pragma unroll
    for (int h = 0; h < 2; ++h) x[h] = *reinterpret_cast<const V8*>(xrow + block * 64 + 32 * h);
  }
  __device__ __forceinline__ void compute(f32x4 (&acc)[1][R]) const {
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int h = 0; h < 2; ++h) acc[0][r] = Mfma16<T>::run(x[h], __builtin_bit_cast(V8, w[r][h]), acc[0][r]);
  }
};

__device__ __forceinline__ float silu_mul(float g, float u) { return g / (1.0f + expf(-g)) * u; }

}  // namespace ember
