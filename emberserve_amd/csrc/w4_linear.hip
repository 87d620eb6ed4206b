// Projections over 4-bit weights with group scales, for the tokens of a decode step:
//   out[t, n] = round(sum_k x[t, k] s[n, g(k)] (q[n, k] - z[n, g(k)]) + bias[n])
// and the dense MLP's gate_up form, round(silu(gate) * up), over the packed layout of w4.h.
//
// What bounds it: the weights' bytes (N K / 2 and the scales), read once. A wave holds R slabs of 16
// weight rows against up to 64 tokens, so a block's codes are loaded once (one 16-byte non-temporal
// load per lane and slab) and turned into MFMA operands in registers; nothing goes through LDS but
// the sums of the waves that share a slab's k.
#include <algorithm>

#include "w4.h"

namespace ember {
namespace {

constexpr int kW4Waves = 8;
constexpr int kW4Tokens = 64;  // tokens of one pass over the weights

struct W4Args {
  const void* x;
  int64_t xs;
  const uint8_t* w;
  const void* bias;
  void* out;
  int64_t os;
  int T, K, N;   // N: columns of out
  int slabs, nb; // slabs of the packed weight (gate_up: twice the column slabs), blocks of k
  int wk;        // waves that share a slab's k: 1, 2, 4 or 8
  int gate_up;
};

// NT token tiles of 16, R slabs a wave, D blocks in flight.
template <typename T, int NT, int R, int GPB, int D>
__global__ void __launch_bounds__(kW4Waves * kWave)
k_w4_linear(W4Args a) {
  using S = Stage<T, R, NT, GPB>;
  extern __shared__ __attribute__((aligned(16))) float red[];  // wk > 1: [wave][NT * R][lane] x 4
  const int lane = threadIdx.x & (kWave - 1);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int kpart = wave & (a.wk - 1);
  const int slab0 = (blockIdx.x * (kW4Waves / a.wk) + wave / a.wk) * R;
  const int tok0 = blockIdx.y * kW4Tokens;
  const uint8_t* base[R];
#pragma unroll
  for (int r = 0; r < R; ++r)
    base[r] = a.w + static_cast<int64_t>(min(slab0 + r, a.slabs - 1)) * a.nb * w4_block_bytes(GPB);
  const T* xrow[NT];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
    xrow[nt] = static_cast<const T*>(a.x) + static_cast<int64_t>(min(tok0 + 16 * nt + (lane & 15), a.T - 1)) * a.xs +
               8 * (lane >> 4);
  S ring[D];
  f32x4 acc[NT][R];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int r = 0; r < R; ++r) acc[nt][r] = f32x4{0.f, 0.f, 0.f, 0.f};
  const int nj = slab0 < a.slabs && kpart < a.nb ? (a.nb - kpart + a.wk - 1) / a.wk : 0;
  auto issue = [&](S& st, int j) {
    const int b = min(kpart + j * a.wk, a.nb - 1);
#pragma unroll
    for (int r = 0; r < R; ++r) st.load_w4(r, base[r], b, lane);
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) st.load_x(nt, xrow[nt], b, a.K);
  };
  if (nj > 0) {
#pragma unroll
    for (int d = 0; d < D; ++d) {
      issue(ring[d], d);
      __builtin_amdgcn_sched_barrier(0);
    }
    int j0 = 0;
    for (; j0 + D < nj; j0 += D) {
#pragma unroll
      for (int d = 0; d < D; ++d) {
        ring[d].compute(acc);
        issue(ring[d], j0 + D + d);
        __builtin_amdgcn_sched_barrier(0);
      }
    }
#pragma unroll
    for (int d = 0; d < D; ++d)
      if (j0 + d < nj) ring[d].compute(acc);
  }

  // lane: column l % 16 of its slab, tokens 16 nt + 4 (l / 16) + i
  auto emit = [&](int nt, int slab, f32x4 v, f32x4 up) {
    const int col = (a.gate_up ? slab >> 1 : slab) * 16 + (lane & 15);
    if (col >= a.N) return;
    const float bias = a.bias != nullptr ? to_f32(static_cast<const T*>(a.bias)[col]) : 0.0f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int tok = tok0 + 16 * nt + 4 * (lane >> 4) + i;
      if (tok >= a.T) continue;
      const float y = a.gate_up ? silu_mul(v[i], up[i]) : v[i] + bias;
      static_cast<T*>(a.out)[static_cast<int64_t>(tok) * a.os + col] = from_f32<T>(y);
    }
  };
  const int step = a.gate_up ? 2 : 1;  // gate and up slabs alternate; R is even then
  if (a.wk == 1) {
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int r = 0; r < R; ++r)
        if ((r % 2 == 0 || step == 1) && slab0 + r < a.slabs) emit(nt, slab0 + r, acc[nt][r], acc[nt][R > 1 ? (r | 1) : 0]);
    return;
  }
  f32x4* lds = reinterpret_cast<f32x4*>(red);
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int r = 0; r < R; ++r) lds[(wave * NT * R + nt * R + r) * kWave + lane] = acc[nt][r];
  __syncthreads();
  // the waves of a slab take its tiles in turn, summing the k parts in order
  const int first = wave - kpart;
  auto total = [&](int tile) {
    f32x4 v = lds[(first * NT * R + tile) * kWave + lane];
    for (int q = 1; q < a.wk; ++q) v += lds[((first + q) * NT * R + tile) * kWave + lane];
    return v;
  };
  for (int tile = kpart * step; tile < NT * R; tile += a.wk * step) {
    const int slab = slab0 + tile % R;
    if (slab >= a.slabs) continue;
    const f32x4 v = total(tile);
    emit(tile / R, slab, v, a.gate_up ? total(tile + 1) : v);
  }
}

template <typename T, int NT, int R, int GPB, int D>
int w4_launch(const W4Args& a, hipStream_t stream) {
  const int groups = static_cast<int>(cdiv(a.slabs, R));
  const dim3 grid(static_cast<unsigned>(cdiv(groups, kW4Waves / a.wk)), static_cast<unsigned>(cdiv(a.T, kW4Tokens)));
  const size_t lds = a.wk > 1 ? size_t(kW4Waves) * NT * R * kWave * 16 : 0;
  k_w4_linear<T, NT, R, GPB, D><<<grid, kW4Waves * kWave, lds, stream>>>(a);
  return launch_status();
}

// Slabs a wave and waves along k, from sizes: see w4_run.
template <typename T, int GPB>
int w4_pick(W4Args a, int r, hipStream_t stream) {
  const int nt = a.T <= 16 ? 1 : (a.T <= 32 ? 2 : 4);
  if (nt == 1) {
    if (r == 1) return w4_launch<T, 1, 1, GPB, 4>(a, stream);
    if (r == 2) return w4_launch<T, 1, 2, GPB, 4>(a, stream);
    return w4_launch<T, 1, 4, GPB, 3>(a, stream);
  }
  if (nt == 2) {
    if (r == 1) return w4_launch<T, 2, 1, GPB, 3>(a, stream);
    if (r == 2) return w4_launch<T, 2, 2, GPB, 3>(a, stream);
    return w4_launch<T, 2, 4, GPB, 2>(a, stream);
  }
  if (r == 1) return w4_launch<T, 4, 1, GPB, 2>(a, stream);
  if (r == 2) return w4_launch<T, 4, 2, GPB, 2>(a, stream);
  return w4_launch<T, 4, 4, GPB, 1>(a, stream);
}

template <typename T>
int w4_run(W4Args a, int gpb, hipStream_t stream) {
  const int64_t waves = 8 * std::max(1, device_cu_count());
  // Slabs a wave: more of them share a block's tokens; as many as leave the chip its waves.
  int r = a.gate_up ? 2 : 1;
  const int most = a.T <= 16 ? 2 : 4;
  while (r < most && a.slabs / (2 * r) >= waves) r *= 2;
  int wk = 1;
  while (wk < kW4Waves && cdiv(a.slabs, r) * wk < waves && 2 * wk <= a.nb) wk *= 2;
  const int nt = a.T <= 16 ? 1 : (a.T <= 32 ? 2 : 4);
  if (wk > 1 && nt * r > 8) wk = 1;  // 64 KiB of LDS
  a.wk = wk;
  switch (gpb) {
    case 1: return w4_pick<T, 1>(a, r, stream);
    case 2: return w4_pick<T, 2>(a, r, stream);
    default: return w4_pick<T, 4>(a, r, stream);
  }
}

bool group_ok(int64_t k, int64_t group) {
  if (group == 32 || group == 64) return k % group == 0;
  return group >= kW4Block && group % kW4Block == 0 && k % group == 0;
}

bool sizes_ok(int64_t rows, int64_t k, int64_t group) {
  return rows >= 1 && rows <= (int64_t(1) << 27) && k >= 32 && k <= (int64_t(1) << 24) && group_ok(k, group);
}

int w4_call(const void* x, int64_t xs, const void* packed, int64_t group, int dtype, int64_t tokens, int64_t k,
            int64_t rows, int gate_up, const void* bias, void* out, int64_t os, void* stream) {
  if (tokens == 0 && sizes_ok(rows, k, group)) return EMBER_OK;
  if (x == nullptr || packed == nullptr || out == nullptr || tokens < 0 || tokens > (int64_t(1) << 21) ||
      !sizes_ok(rows, k, group) || (dtype != EMBER_F16 && dtype != EMBER_BF16) || os < 0 || xs < 0)
    return EMBER_EINVAL;
  if (!aligned16(x) || !aligned16(packed) || xs % 8 != 0) return EMBER_EALIGN;
  W4Args a{x, xs, static_cast<const uint8_t*>(packed), bias, out, os, static_cast<int>(tokens), static_cast<int>(k),
           static_cast<int>(rows), static_cast<int>(cdiv(rows, 16)) * (gate_up ? 2 : 1),
           static_cast<int>(cdiv(k, kW4Block)), 1, gate_up};
  const int gpb = w4_gpb(group);
  hipStream_t s = static_cast<hipStream_t>(stream);
  return dtype == EMBER_F16 ? w4_run<_Float16>(a, gpb, s) : w4_run<__bf16>(a, gpb, s);
}

// ---- packing ----------------------------------------------------------------------------

struct W4PackArgs {
  const uint8_t* codes;
  int64_t ces, crs;
  const void* scales;
  int64_t ses, srs;
  int scale_dtype;
  const uint8_t* zeros;
  int64_t zes, zrs;
  int rows, k, group, parts, gpb, nb;
  uint8_t* dst;
  int64_t pieces;  // 16-byte pieces in all
};

// One 16-byte piece of the packed array a thread: lane `lane`'s codes of a block, or four scales.
__global__ void __launch_bounds__(256) k_w4_pack(W4PackArgs a) {
  const int per = 64 + 4 * a.gpb;  // pieces of a block
  const int slabs = (a.rows + 15) / 16 * a.parts;
  for (int64_t t = int64_t(blockIdx.x) * 256 + threadIdx.x; t < a.pieces; t += int64_t(gridDim.x) * 256) {
    int64_t q = t / per;
    const int piece = static_cast<int>(t - q * per);
    const int b = static_cast<int>(q % a.nb);
    q /= a.nb;
    const int s = static_cast<int>(q % slabs);
    const int64_t e = q / slabs;
    const int row0 = s / a.parts * 16;             // first row within the part
    const int64_t part = int64_t(s % a.parts) * a.rows;
    u32x4 v = {0, 0, 0, 0};
    if (piece < 64) {
      const int row = row0 + (piece & 15);
      if (row < a.rows) {
        const uint8_t* src = a.codes + e * a.ces + (part + row) * a.crs;
        for (int f = 0; f < 4; ++f) {
          const int k0 = kW4Block * b + 32 * f + 8 * (piece >> 4);
          if (k0 >= a.k) continue;
          uint32_t w = 0;
          for (int i = 0; i < 4; ++i) {  // byte i: codes 2 i (low nibble) and 2 i + 1
            const uint32_t c = src[k0 / 2 + i];
            w |= (c & 15u) << (4 * i) | (c >> 4) << (16 + 4 * i);
          }
          v[f] = w;
        }
      }
    } else {
      for (int i = 0; i < 4; ++i) {
        const int word = (piece - 64) * 4 + i;  // [row][gpb]
        const int row = row0 + word / a.gpb;
        const int k0 = kW4Block * b + word % a.gpb * (kW4Block / a.gpb);
        if (row >= a.rows || k0 >= a.k) continue;
        const int g = k0 / a.group;
        const int64_t at = e * a.ses + (part + row) * a.srs + g;
        const float sc = a.scale_dtype == EMBER_F16 ? to_f32(static_cast<const _Float16*>(a.scales)[at])
                                                    : to_f32(static_cast<const __bf16*>(a.scales)[at]);
        const uint32_t z = a.zeros != nullptr ? a.zeros[e * a.zes + (part + row) * a.zrs + g] & 15u : 8u;
        v[i] = (__builtin_bit_cast(uint32_t, sc) & ~15u) | z;
      }
    }
    *reinterpret_cast<u32x4*>(a.dst + t * 16) = v;
  }
}

}  // namespace
}  // namespace ember

using namespace ember;

extern "C" {

int64_t ember_w4_packed_bytes(int64_t rows, int64_t k, int64_t group, int gate_up) {
  if (!sizes_ok(rows, k, group)) return -1;
  return cdiv(rows, 16) * (gate_up ? 2 : 1) * cdiv(k, kW4Block) * w4_block_bytes(w4_gpb(group));
}

int ember_w4_pack_weight(const void* codes, int64_t code_expert_stride, int64_t code_row_stride, const void* scales,
                         int64_t scale_expert_stride, int64_t scale_row_stride, int scale_dtype, const void* zeros,
                         int64_t zero_expert_stride, int64_t zero_row_stride, int64_t num_experts, int64_t rows,
                         int64_t k, int64_t group, int gate_up, void* packed, void* stream) {
  const int64_t bytes = ember_w4_packed_bytes(rows, k, group, gate_up);
  if (codes == nullptr || scales == nullptr || packed == nullptr || num_experts < 1 || bytes < 0 ||
      num_experts > INT64_MAX / bytes || (scale_dtype != EMBER_F16 && scale_dtype != EMBER_BF16))
    return EMBER_EINVAL;
  if (!aligned16(packed)) return EMBER_EALIGN;
  W4PackArgs a{static_cast<const uint8_t*>(codes), code_expert_stride, code_row_stride, scales, scale_expert_stride,
               scale_row_stride, scale_dtype, static_cast<const uint8_t*>(zeros), zero_expert_stride, zero_row_stride,
               static_cast<int>(rows), static_cast<int>(k), static_cast<int>(std::min<int64_t>(group, k)),
               gate_up ? 2 : 1, w4_gpb(group), static_cast<int>(cdiv(k, kW4Block)), static_cast<uint8_t*>(packed),
               num_experts * bytes / 16};
  const int64_t grid = std::min<int64_t>(cdiv(a.pieces, 256), 65536);
  k_w4_pack<<<dim3(static_cast<unsigned>(grid)), 256, 0, static_cast<hipStream_t>(stream)>>>(a);
  return launch_status();
}

int ember_w4_linear(const void* x, int64_t x_row_stride, const void* packed, int64_t group, int dtype, int64_t tokens,
                    int64_t k, int64_t rows, const void* bias, void* out, int64_t out_row_stride, void* stream) {
  return w4_call(x, x_row_stride, packed, group, dtype, tokens, k, rows, 0, bias, out, out_row_stride, stream);
}

int ember_w4_gate_up_silu(const void* x, int64_t x_row_stride, const void* packed, int64_t group, int dtype,
                          int64_t tokens, int64_t hidden, int64_t inter, void* out, int64_t out_row_stride,
                          void* stream) {
  return w4_call(x, x_row_stride, packed, group, dtype, tokens, hidden, inter, 1, nullptr, out, out_row_stride, stream);
}

}  // extern "C"
