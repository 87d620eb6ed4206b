// Projections over 4-bit weights with group scales, for the tokens of a decode step:
//   out[t, n] = round(sum_k x[t, k] s[n, g(k)] (q[n, k] - z[n, g(k)]) + bias[n])
// and the dense MLP's gate_up form, round(silu(gate) * up), over the packed layout of w4.h.
//
// What bounds it: the weights' bytes (N K / 2 and the scales), read once, and what a CU can issue of loads:
// the tokens are loaded again by every workgroup (from L2). A wave holds 1 to 4 slabs of 16 weight rows
// against up to 32 tokens; a block of 128 k of a slab is one 16-byte non-temporal load a lane, turned into
// MFMA operands in registers.
#include <algorithm>

#include "w4.h"

namespace ember {
namespace {

struct W4Args {
  const void* x;
  int64_t xs;
  const uint8_t* w;
  const void* bias;
  void* out;
  int64_t os;
  int T, K, N;   // N: columns of out
  int slabs, nb; // slabs of the packed weight (gate_up: twice the column slabs), blocks of k
  int groups;    // sets of R slabs
  int tiles;     // sets of 16 NT tokens
  int gate_up;
  int side;      // k_w4_wide: waves side by side
  int splits;    // k_w4_linear: workgroups that share a set's k, ...
  float* part;   // ... their sums [group][tile][split][nt R + r][lane][4] (null: no splits)
  uint32_t* counters;  // and arrivals [group][tile]
};

constexpr int kXcds = 8;
constexpr int kW4MaxSplits = 8;
constexpr int kSplitTokens = 64;  // most tokens whose k is split: more fill the chip

// A workgroup holds R slabs against NT tiles of 16 tokens (XI < 4: of 4 XI); its waves, and those of the
// other splits, share k, block by block. D blocks in flight a wave.
template <typename T, int R, int GPB, int NT, int XI, int D, int MAXW>
__global__ void __launch_bounds__(MAXW * kWave)
k_w4_linear(W4Args a) {
  using X = XBlock<NT, XI>;
  constexpr int P = X::kPieces > 64 * R * NT ? X::kPieces : 64 * R * NT;
  extern __shared__ __attribute__((aligned(16))) u32x4 lds[];  // [wave][P]: a block's tokens, then the sums
  __shared__ int last;
  const int lane = threadIdx.x & (kWave - 1);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wk = blockDim.x >> 6;
  // the tiles of a slab group on one XCD, next to each other: its L2 holds the weights for them
  const int per = kXcds * a.tiles * a.splits;
  const int sub = blockIdx.x % per / kXcds;
  const int split = a.splits > 1 ? sub / a.tiles : 0, tile = sub - split * a.tiles;
  const int first = split * wk + wave, stride = a.splits * wk;
  const int group = blockIdx.x / per * kXcds + blockIdx.x % kXcds;
  if (group >= a.groups) return;
  const int slab0 = group * R, tok0 = 16 * NT * tile;
  const int rows = min(a.T - tok0, 16 * NT);
  const BufferRsrc xr = buffer(static_cast<const T*>(a.x) + static_cast<int64_t>(tok0) * a.xs,
                               static_cast<int>(((rows - 1) * a.xs + a.K) * 2));
  int off[NT * XI];
#pragma unroll
  for (int i = 0; i < NT * XI; ++i)
    off[i] = min(4 * i + (lane >> 4), rows - 1) * static_cast<int>(a.xs) * 2 + 16 * (lane & 15);
  const int64_t slab_bytes = w4_slab_bytes(a.nb, GPB);
  BufferRsrc base[R];
#pragma unroll
  for (int r = 0; r < R; ++r)
    base[r] = buffer(a.w + min(slab0 + r, a.slabs - 1) * slab_bytes, static_cast<int>(slab_bytes));

  struct Stage {
    W4Block<R, GPB> w;
    X x;
  };
  u32x4* const mine = lds + wave * P;
  f32x4 acc[NT][R];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int r = 0; r < R; ++r) acc[nt][r] = f32x4{0.f, 0.f, 0.f, 0.f};
  stream<Stage, D>(
      0, first < a.nb ? (a.nb - first + stride - 1) / stride : 0,
      [&](Stage& g, int j) {
        const int b = min(first + j * stride, a.nb - 1);
#pragma unroll
        for (int r = 0; r < R; ++r) g.w.load(r, base[r], b, a.nb, lane);
        g.x.load(xr, off, b, a.K, lane);
      },
      [&](const Stage& g, int) {
        g.x.put(mine, lane);
        g.w.template compute<T, NT>([&](int nt, int f) { return X::frag(mine, nt, f, lane); }, acc);
      });

  // lane: column l % 16 of its slab, tokens 16 nt + 4 (l / 16) + i
  auto emit = [&](int nt, int slab, f32x4 v, f32x4 up) {
    const int col = (a.gate_up ? slab >> 1 : slab) * 16 + (lane & 15);
    if (slab >= a.slabs || col >= a.N) return;
    const float bias = a.bias != nullptr ? to_f32(static_cast<const T*>(a.bias)[col]) : 0.0f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int tok = 16 * nt + 4 * (lane >> 4) + i;
      if (tok >= rows) continue;
      const float y = a.gate_up ? silu_mul(v[i], up[i]) : v[i] + bias;
      static_cast<T*>(a.out)[static_cast<int64_t>(tok0 + tok) * a.os + col] = from_f32<T>(y);
    }
  };
  if (wk == 1 && a.splits == 1) {
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int r = 0; r < R; ++r)
        if (r % 2 == 0 || !a.gate_up) emit(nt, slab0 + r, acc[nt][r], acc[nt][(r | 1) < R ? r | 1 : r]);
    return;
  }
  // the waves take the tiles (gate and up together) in turn, summing the waves' shares of k in order
  f32x4* const red = reinterpret_cast<f32x4*>(lds);
  asm volatile("" ::: "memory");
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int r = 0; r < R; ++r) red[wave * P + (nt * R + r) * kWave + lane] = acc[nt][r];
  __syncthreads();
  auto total = [&](int t) {
    f32x4 v = red[t * kWave + lane];
    for (int q = 1; q < wk; ++q) v += red[q * P + t * kWave + lane];
    return v;
  };
  if (a.splits > 1) {  // not gate_up
    const int set = group * a.tiles + tile;
    constexpr int kSums = NT * R * kWave;
    const CoherentRsrc rs =
        coherent_rsrc(a.part + static_cast<int64_t>(set) * a.splits * kSums * 4, a.splits * kSums * 4);
    for (int t = wave; t < NT * R; t += wk) store_coherent<4>(rs, (split * kSums + t * kWave + lane) * 16, total(t));
    __builtin_amdgcn_s_waitcnt(0);
    __syncthreads();
    if (threadIdx.x == 0) {
      const uint32_t prev = __hip_atomic_fetch_add(a.counters + set, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      last = prev == static_cast<uint32_t>(a.splits) - 1;
      if (last) __hip_atomic_store(a.counters + set, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    __syncthreads();
    if (!last) return;
    for (int t = wave; t < NT * R; t += wk) {  // in the splits' order, whoever is last
      f32x4 v[kW4MaxSplits];
#pragma unroll
      for (int s = 0; s < kW4MaxSplits; ++s)
        v[s] = load_coherent<4>(rs, (min(s, a.splits - 1) * kSums + t * kWave + lane) * 16);
      f32x4 y = v[0];
#pragma unroll
      for (int s = 1; s < kW4MaxSplits; ++s) y += s < a.splits ? v[s] : f32x4{0.f, 0.f, 0.f, 0.f};
      emit(t / R, slab0 + t % R, y, y);
    }
    return;
  }
  const int step = a.gate_up ? 2 : 1;
  for (int t = wave * step; t < NT * R; t += wk * step) {
    const f32x4 v = total(t);
    emit(t / R, slab0 + t % R, v, a.gate_up ? total(t + 1) : v);
  }
}

// Many slabs: G waves side by side, of R slabs each, share every block's tokens through LDS, in WK such
// teams along k. A CU takes in about 10 bytes a clock whether they come from memory or L2 (6.4 TB/s over
// all), so that the tokens count like weights: at 27 tokens and 4 slabs a workgroup they were twice the
// weights' bytes. Each wave loads XS of a block's 4 NT pieces of 4 rows, D blocks ahead with its weights,
// and puts them into LDS; one barrier a block, two buffers a team.
constexpr int kWideWaves = 12;
constexpr int kWideLds = 65536;

template <typename T, int GPB, int NT, int XS, int D>
__global__ void __launch_bounds__(kWideWaves * kWave)
k_w4_wide(W4Args a) {
  constexpr int R = 2;
  extern __shared__ __attribute__((aligned(16))) u32x4 lds[];  // [team][2][256 NT], then the teams' sums
  const int lane = threadIdx.x & (kWave - 1);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int side = a.side, wk = (blockDim.x >> 6) / side;
  const int team = wave / side, place = wave - team * side;
  const int group = blockIdx.x * side + place;
  const int slab0 = group * R, tok0 = 16 * NT * blockIdx.y;
  const bool real = group < a.groups;  // the last workgroup's other waves only help with the tokens
  const int rows = min(a.T - tok0, 16 * NT);
  const BufferRsrc xr = buffer(static_cast<const T*>(a.x) + static_cast<int64_t>(tok0) * a.xs,
                               static_cast<int>(((rows - 1) * a.xs + a.K) * 2));
  int off[XS];
#pragma unroll
  for (int i = 0; i < XS; ++i)
    off[i] = min(4 * (place + i * side) + (lane >> 4), rows - 1) * static_cast<int>(a.xs) * 2 + 16 * (lane & 15);
  const int64_t slab_bytes = w4_slab_bytes(a.nb, GPB);
  BufferRsrc base[R];
#pragma unroll
  for (int r = 0; r < R; ++r)
    base[r] = buffer(a.w + min(slab0 + r, a.slabs - 1) * slab_bytes, static_cast<int>(slab_bytes));

  struct Stage {
    W4Block<R, GPB> w;
    u32x4 x[XS];
  };
  f32x4 acc[NT][R];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int r = 0; r < R; ++r) acc[nt][r] = f32x4{0.f, 0.f, 0.f, 0.f};
  stream<Stage, D>(
      0, (a.nb + wk - 1) / wk,  // the same for all waves: the barriers
      [&](Stage& g, int j) {
        const int b = min(team + j * wk, a.nb - 1);
#pragma unroll
        for (int r = 0; r < R; ++r) g.w.load(r, base[r], b, a.nb, lane);
        const int past = nowhere(b * kW4Block + 8 * (lane & 15) >= a.K);
#pragma unroll
        for (int i = 0; i < XS; ++i) g.x[i] = __builtin_amdgcn_raw_buffer_load_b128(xr, off[i] | past, b * (2 * kW4Block), 0);
      },
      [&](const Stage& g, int j) {
        u32x4* const x = lds + (team * 2 + (j & 1)) * (256 * NT);
#pragma unroll
        for (int i = 0; i < XS; ++i) {
          const int r = 4 * (place + i * side) + (lane >> 4);
          if (r < 16 * NT) x[16 * r + ((lane & 15) ^ (r & 15))] = g.x[i];
        }
        lds_barrier();
        if (real && team + j * wk < a.nb)
          g.w.template compute<T, NT>([&](int nt, int f) { return XBlock<NT, 4>::frag(x, nt, f, lane); }, acc);
      });

  // lane: column l % 16 of its slab, tokens 16 nt + 4 (l / 16) + i
  f32x4* const red = reinterpret_cast<f32x4*>(lds) + place * (NT * R * kWave);
  const int each = side * NT * R * kWave;
  if (wk > 1) {
    __syncthreads();
    if (team > 0) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int r = 0; r < R; ++r) red[(team - 1) * each + (nt * R + r) * kWave + lane] = acc[nt][r];
    }
    __syncthreads();
  }
  if (team > 0 || !real) return;
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
    for (int r = 0; r < R; ++r)
      for (int q = 0; q < wk - 1; ++q) acc[nt][r] += red[q * each + (nt * R + r) * kWave + lane];
    auto put = [&](int slab, f32x4 v, f32x4 up) {
      const int col = (a.gate_up ? slab >> 1 : slab) * 16 + (lane & 15);
      if (slab >= a.slabs || col >= a.N) return;
      const float bias = a.bias != nullptr ? to_f32(static_cast<const T*>(a.bias)[col]) : 0.0f;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int tok = 16 * nt + 4 * (lane >> 4) + i;
        if (tok >= rows) continue;
        const float y = a.gate_up ? silu_mul(v[i], up[i]) : v[i] + bias;
        static_cast<T*>(a.out)[static_cast<int64_t>(tok0 + tok) * a.os + col] = from_f32<T>(y);
      }
    };
    put(slab0, acc[nt][0], acc[nt][1]);
    if (!a.gate_up) put(slab0 + 1, acc[nt][1], acc[nt][1]);
  }
}

template <typename T, int GPB, int NT, int XS, int D>
int wide_launch(W4Args a, int wk, hipStream_t stream) {
  const size_t lds = std::max<size_t>(size_t(wk) * 2 * 4096 * NT, size_t(wk - 1) * a.side * NT * 2048);
  const dim3 grid(static_cast<unsigned>(cdiv(a.groups, a.side)), static_cast<unsigned>(cdiv(a.T, 16 * NT)));
  k_w4_wide<T, GPB, NT, XS, D><<<grid, a.side * wk * kWave, lds, stream>>>(a);
  return launch_status();
}

// Waves side by side, for 9 tokens and more: the pairs of slabs that each CU gets, where that is 2 to 8 (one
// round of workgroups). Measured (us, k_w4_linear | k_w4_wide): gate_up 768 pairs x 4096, 8 tokens 14.2 |
// 15.2, 16: 16.6 | 15.9, 32: 21.3 | 19.8, 64 (two passes of 32 with 3 waves side by side) 28.5 | 37.2; 1184
// pairs x 3584, 16: 23.0 | 19.4, 32: 28.6 | 24.8, 64: 42.2 | 35.2; the head's 4748 pairs x 4096, 16: 69.3 | 77.
int wide_side(const W4Args& a) {
  const int64_t cus = std::max(1, device_cu_count()), pairs = cdiv(a.slabs, 2), side = cdiv(pairs, cus);
  if (a.T <= 8 || side > 8 || 4 * pairs < 7 * cus || (a.T > 32 && side < 4)) return 0;
  return static_cast<int>(side);
}

template <typename T, int GPB>
int wide_pick(W4Args a, hipStream_t stream) {
  const bool most = a.side >= 4;
  const int nt = a.T <= 16 ? 1 : (a.T <= 32 ? 2 : 4);
  int wk = kWideWaves / a.side;
  while (wk > 1 && (wk * 8192 * nt > kWideLds || (wk - 1) * a.side * nt * 2048 > kWideLds || 2 * wk > a.nb)) --wk;
  if (nt == 1) return most ? wide_launch<T, GPB, 1, 1, 4>(a, wk, stream) : wide_launch<T, GPB, 1, 2, 4>(a, wk, stream);
  if (nt == 2) return most ? wide_launch<T, GPB, 2, 2, 4>(a, wk, stream) : wide_launch<T, GPB, 2, 4, 3>(a, wk, stream);
  return wide_launch<T, GPB, 4, 4, 2>(a, wk, stream);
}

template <typename T, int R, int GPB, int NT, int XI, int D, int MAXW>
int w4_launch(W4Args a, hipStream_t stream) {
  const int64_t cus = std::max(1, device_cu_count());
  a.groups = static_cast<int>(cdiv(a.slabs, R));
  a.tiles = static_cast<int>(cdiv(a.T, 16 * NT));
  const int64_t grid = cdiv(a.groups, kXcds) * kXcds * a.tiles * a.splits;
  // Waves along k: 7 or more a CU, each with at least a block or two. Measured (us): Qwen2.5-7B down, 2
  // tokens (224 slabs, 148 blocks) 12.6 with 4, 11.8 with 8, 13.6 with 16; Qwen3-8B head, 16 tokens (2374
  // sets of slabs) 70.4 with 1, 75.6 with 2.
  int wk = 1;
  while (wk < MAXW && grid * wk < 7 * cus && 2 * wk * a.splits < a.nb) wk *= 2;
  const size_t lds = size_t(wk) * 16 * std::max(XBlock<NT, XI>::kPieces, 64 * R * NT);
  k_w4_linear<T, R, GPB, NT, XI, D, MAXW><<<dim3(static_cast<unsigned>(grid)), wk * kWave, lds, stream>>>(a);
  return launch_status();
}

// Slabs a workgroup and splits of k. More slabs share a block's tokens, but fewer workgroups fill the chip,
// unless several split the slabs' k and join their sums. The choice with the shortest rounds: a block is 1 KiB
// a slab at the 24 GB/s that a CU takes in from memory, and XI NT KiB of tokens at three times that from L2;
// a join costs 3 us, what 80 KiB from memory do. Splits that only even out the last round lose: the head's 9496
// slabs x 4096, 16 tokens 4/1 64.5, 4/2 82.6. Measured (us at slabs/splits): 256 slabs x 4096, 16 tokens
// 1/1 7.5, 2/1 8.6, 4/4 9.7; 384 x 4096, 16 tokens 2/1 8.0, 1/1 10.3, 61 tokens 3/1 12.3, 4/1 13.1, 2/2 15.1;
// 224 x 18944, 6 tokens 1/1 13.1, 4/4 13.4, 16 tokens 4/4 14.9, 1/1 16.9, 24 tokens 4/4 17.1, 2/2 18.9, 1/1 23.7,
// 61 tokens 4/2 25.3, 2/1 29.0; gate_up 1536 x 4096, 16 tokens 2/1 18.3, 4/1 21.9, 64 tokens 4/1 31.6, 2/1 35.1.
struct W4Shape {
  int r, splits;
};
W4Shape w4_shape(const W4Args& a, int nt, int xi, bool split) {
  const int64_t cus = std::max(1, device_cu_count()), tiles = cdiv(a.T, 16 * nt);
  W4Shape best{0, 1};
  int64_t least = 0;
  for (int s = 1; s == 1 || (split && s <= kW4MaxSplits && 8 * s <= a.nb); ++s)
    for (int r = a.gate_up ? 2 : 1; r <= 4; r += a.gate_up ? 2 : 1) {
      const int64_t wgs = cdiv(a.slabs, r) * tiles * s;
      if (s > 1 && wgs > 2 * cus) continue;  // the chip is full without
      const int64_t cost =
          cdiv(wgs, cus) * cdiv(a.nb, s) * (3 * r + xi * nt) + (s > 1 ? 3 * 80 : 0);
      if (best.r == 0 || cost < least) {
        best = {r, s};
        least = cost;
      }
    }
  return best;
}
// The same of a call, for w4_pick and for the size of its workspace.
W4Shape w4_shape(const W4Args& a, bool split) {
  return w4_shape(a, a.T <= 16 ? 1 : 2, a.T <= 8 ? 2 : 4, split && !a.gate_up && a.T <= kSplitTokens);
}

// Token tiles, slabs and depth by size. Two tiles a wave from 17 tokens: the codes are turned into operands
// once for both (gate_up of Qwen2.5-7B, 27 tokens, 35.6 us with one tile a wave, 28.8 with two). Up to 4
// and 8 tokens a block's tokens are one and two loads instead of four, and the ring is deeper.
template <typename T, int GPB>
int w4_pick(W4Args a, hipStream_t stream) {
  if (a.T <= 4) {
    if (!a.gate_up) return w4_launch<T, 1, GPB, 1, 1, GPB == 4 ? 6 : 8, 16>(a, stream);
    return w4_launch<T, 2, GPB, 1, 1, GPB == 4 ? 3 : 4, 16>(a, stream);
  }
  if (const int side = wide_side(a); side != 0) {
    a.groups = static_cast<int>(cdiv(a.slabs, 2));
    a.side = side;
    return wide_pick<T, GPB>(a, stream);
  }
  const W4Shape shape = w4_shape(a, a.part != nullptr);
  const int r = shape.r;
  a.splits = shape.splits;
  if (a.T <= 8) {
    if (r == 1) return w4_launch<T, 1, GPB, 1, 2, 4, 16>(a, stream);
    if (r == 2) return w4_launch<T, 2, GPB, 1, 2, 4, 8>(a, stream);
    if (r == 3) return w4_launch<T, 3, GPB, 1, 2, 3, 8>(a, stream);
    return w4_launch<T, 4, GPB, 1, 2, 3, 8>(a, stream);
  }
  if (a.T <= 16) {
    if (r == 1) return w4_launch<T, 1, GPB, 1, 4, GPB == 1 ? 4 : 3, 16>(a, stream);
    if (r == 2) return w4_launch<T, 2, GPB, 1, 4, 4, 8>(a, stream);
    if (r == 3) return w4_launch<T, 3, GPB, 1, 4, 3, 8>(a, stream);
    return w4_launch<T, 4, GPB, 1, 4, 3, 8>(a, stream);
  }
  if (r == 1) return w4_launch<T, 1, GPB, 2, 4, 3, 8>(a, stream);
  if (r == 2) return w4_launch<T, 2, GPB, 2, 4, 2, 8>(a, stream);
  if (r == 3) return w4_launch<T, 3, GPB, 2, 4, 2, 8>(a, stream);
  return w4_launch<T, 4, GPB, 2, 4, 2, 8>(a, stream);
}

template <typename T>
int w4_run(const W4Args& a, int gpb, hipStream_t stream) {
  switch (gpb) {
    case 1: return w4_pick<T, 1>(a, stream);
    case 2: return w4_pick<T, 2>(a, stream);
    default: return w4_pick<T, 4>(a, stream);
  }
}

bool group_ok(int64_t k, int64_t group) {
  if (group == 32 || group == 64) return k % group == 0;
  return group >= kW4Block && group % kW4Block == 0 && k % group == 0;
}

bool sizes_ok(int64_t rows, int64_t k, int64_t group) {
  return rows >= 1 && rows <= (int64_t(1) << 27) && k >= 32 && k <= (int64_t(1) << 24) && group_ok(k, group);
}

struct W4Space {
  int64_t part, counters;  // bytes
};
// What a call's splits need: nothing for most.
W4Space w4_space(const W4Args& a) {
  if (a.T <= 4 || a.T > kSplitTokens || a.gate_up || wide_side(a) != 0) return {0, 0};
  const W4Shape s = w4_shape(a, true);
  if (s.splits == 1) return {0, 0};
  const int nt = a.T <= 16 ? 1 : 2;
  const int64_t sets = cdiv(a.slabs, s.r) * cdiv(a.T, 16 * nt);
  return {sets * s.splits * nt * s.r * kWave * 16, cdiv(sets * 4, 256) * 256};
}

W4Args w4_args(int64_t tokens, int64_t k, int64_t rows, int gate_up) {
  W4Args a{};
  a.T = static_cast<int>(tokens);
  a.K = static_cast<int>(k);
  a.N = static_cast<int>(rows);
  a.slabs = static_cast<int>(cdiv(rows, 16)) * (gate_up ? 2 : 1);
  a.nb = static_cast<int>(cdiv(k, kW4Block));
  a.tiles = a.splits = 1;
  a.gate_up = gate_up;
  return a;
}

int w4_call(const void* x, int64_t xs, const void* packed, int64_t group, int dtype, int64_t tokens, int64_t k,
            int64_t rows, int gate_up, const void* bias, void* workspace, int64_t workspace_bytes, void* out,
            int64_t os, void* stream) {
  if (tokens == 0 && sizes_ok(rows, k, group)) return EMBER_OK;
  if (x == nullptr || packed == nullptr || out == nullptr || tokens < 0 || tokens > (int64_t(1) << 21) ||
      !sizes_ok(rows, k, group) || xs > (int64_t(1) << 23) || (dtype != EMBER_F16 && dtype != EMBER_BF16) || os < 0 || xs < 0)
    return EMBER_EINVAL;
  if (!aligned16(x) || !aligned16(packed) || xs % 8 != 0) return EMBER_EALIGN;
  W4Args a = w4_args(tokens, k, rows, gate_up);
  a.xs = xs;
  a.w = static_cast<const uint8_t*>(packed);
  a.bias = bias;
  a.os = os;
  if (workspace != nullptr) {
    if (!aligned16(workspace) || workspace_bytes % 16 != 0) return EMBER_EALIGN;
    const W4Space need = w4_space(a);
    if (workspace_bytes < need.part + need.counters) return EMBER_EINVAL;
    if (need.part > 0) {
      a.part = static_cast<float*>(workspace);
      a.counters = reinterpret_cast<uint32_t*>(static_cast<uint8_t*>(workspace) + workspace_bytes - need.counters);
    }
  }
  const int gpb = w4_gpb(group);
  hipStream_t s = static_cast<hipStream_t>(stream);
  // A launch has at most 2^31 threads: a wave for each slab and 16 tokens, where there are so many.
  const int64_t most = std::max<int64_t>(1, (int64_t(1) << 25) / (a.slabs + kXcds)) * 16;
  for (int64_t done = 0; done < tokens; done += most) {
    a.x = static_cast<const uint16_t*>(x) + done * xs;
    a.out = static_cast<uint16_t*>(out) + done * os;
    a.T = static_cast<int>(std::min(most, tokens - done));
    const int st = dtype == EMBER_F16 ? w4_run<_Float16>(a, gpb, s) : w4_run<__bf16>(a, gpb, s);
    if (st != EMBER_OK) return st;
  }
  return EMBER_OK;
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

// One 16-byte piece of the packed array a thread: lane `lane`'s codes of a block, or four words of scales.
__global__ void __launch_bounds__(256) k_w4_pack(W4PackArgs a) {
  const int64_t per = w4_slab_bytes(a.nb, a.gpb) / 16;  // pieces of a slab
  const int slabs = (a.rows + 15) / 16 * a.parts;
  for (int64_t t = int64_t(blockIdx.x) * 256 + threadIdx.x; t < a.pieces; t += int64_t(gridDim.x) * 256) {
    const int64_t sl = t / per;
    const int piece = static_cast<int>(t - sl * per);
    const int64_t e = sl / slabs;
    const int s = static_cast<int>(sl - e * slabs);
    const int row0 = s / a.parts * 16;  // first row within the part
    const int64_t part = int64_t(s % a.parts) * a.rows;
    u32x4 v = {0, 0, 0, 0};
    if (piece < 64 * a.nb) {
      const int lane = piece & 63, row = row0 + (lane & 15);
      if (row < a.rows) {
        const uint8_t* src = a.codes + e * a.ces + (part + row) * a.crs;
        for (int f = 0; f < 4; ++f) {
          const int k0 = kW4Block * (piece >> 6) + 32 * f + 8 * (lane >> 4);
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
        const int word = (piece - 64 * a.nb) * 4 + i;  // [block][row][gpb]
        const int row = row0 + word / a.gpb % 16;
        const int k0 = kW4Block * (word / (16 * a.gpb)) + word % a.gpb * (kW4Block / a.gpb);
        if (row >= a.rows || k0 >= a.k) continue;
        const int64_t at = e * a.ses + (part + row) * a.srs + k0 / a.group;
        const float sc = a.scale_dtype == EMBER_F16 ? to_f32(static_cast<const _Float16*>(a.scales)[at])
                                                    : to_f32(static_cast<const __bf16*>(a.scales)[at]);
        const uint32_t z =
            a.zeros != nullptr ? a.zeros[e * a.zes + (part + row) * a.zrs + k0 / a.group] & 15u : 8u;
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
  return cdiv(rows, 16) * (gate_up ? 2 : 1) * w4_slab_bytes(cdiv(k, kW4Block), w4_gpb(group));
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
  return w4_call(x, x_row_stride, packed, group, dtype, tokens, k, rows, 0, bias, nullptr, 0, out, out_row_stride, stream);
}

int64_t ember_w4_linear_workspace_bytes(int64_t tokens, int64_t k, int64_t rows, int64_t group, int64_t* counter_bytes) {
  if (tokens < 0 || tokens > (int64_t(1) << 21) || !sizes_ok(rows, k, group)) return -1;
  const W4Space s = w4_space(w4_args(tokens, k, rows, 0));
  if (counter_bytes != nullptr) *counter_bytes = s.counters;
  return s.part + s.counters;
}

int ember_w4_linear_split(const void* x, int64_t x_row_stride, const void* packed, int64_t group, int dtype,
                          int64_t tokens, int64_t k, int64_t rows, const void* bias, void* workspace,
                          int64_t workspace_bytes, void* out, int64_t out_row_stride, void* stream) {
  return w4_call(x, x_row_stride, packed, group, dtype, tokens, k, rows, 0, bias, workspace, workspace_bytes, out,
                 out_row_stride, stream);
}

int ember_w4_gate_up_silu(const void* x, int64_t x_row_stride, const void* packed, int64_t group, int dtype,
                          int64_t tokens, int64_t hidden, int64_t inter, void* out, int64_t out_row_stride,
                          void* stream) {
  return w4_call(x, x_row_stride, packed, group, dtype, tokens, hidden, inter, 1, nullptr, nullptr, 0, out, out_row_stride,
                 stream);
}

}  // extern "C"
