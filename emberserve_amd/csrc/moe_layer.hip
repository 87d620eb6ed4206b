// The routed experts' whole layer for a decode step's tokens, in two kernels:
//   act[a, j] = round(silu(x[t] . W1[e, j]) * (x[t] . W1[e, I + j]))     a = t * top_k + c, e = ids[t, c]
//   out[t, n] = round(sum_c weights[t, c] * (W2[e, n] . act[a]))
// (fused_moe_forward, emberserve/model/moe_triton.py:332-345), over fp16/bf16 experts, unpacked or
// packed, and over 4-bit experts (w4.h). g, u and the routed sum stay in fp32; act is rounded once, to be
// an MFMA operand: half a step of the type on each of I terms, which at random signs adds as much to the
// mean error of out as its own rounding does (bf16: 2.4e-3 of the rms, 1.7e-3 from the last rounding alone).
//
// What bounds it: the weights of the experts that the step's tokens reach, each read once. The
// assignments of an expert form groups, of up to 16 (an MFMA tile); 4-bit weights take groups of 4 or 8
// where the mean is small. Every workgroup of the first kernel finds its group in the routing ids by
// itself, so there is no alignment launch: up to 64 assignments, one a lane, by comparing lanes; else by
// a count in LDS. Its waves share the group's k for 16 gate and 16 up rows and meet in LDS; over 4-bit
// weights and enough groups they take 8 column slabs side by side instead, the group's tokens in LDS once.
//
// The second kernel's workgroups hold 16 (4 bits: 32) output columns each for all groups, times a split of
// the work: the waves cut the (group, k block) items of their columns into equal runs, whatever expert
// they belong to, and add each group's finished tile, weighted, to their own fp32 sums [token][column] in
// LDS. The sums of the waves, then of the splits (by the last to arrive, in batches of 16-byte loads: one
// load at a time took 20 us of 52 at 33 tokens), are added in order, so that results do not depend on
// which wave was first.
//
// Measured (Moonlight, 64 experts top-6 of 2048 x 1408, us, first | second kernel): one token 16 | 11,
// 9 tokens 62-68 | 36, 48 tokens 109 | 59 (1047 MB at 6.0 TB/s in all); 4 bits, one token 11 | 9, most of it
// the chain of dependent loads (ids, weights; lists, weights, partials); 128 experts top-8 of 2048 x 768,
// 4 bits, 33 tokens 45 | 29 (268 MB at 3.6 TB/s: the products' issue beside the stream).
#include <algorithm>

#include "w4.h"

namespace ember {
namespace {

constexpr int kMlTile = 16;             // most assignments of a group
constexpr int kMlMaxTokens = 64;
constexpr int kMlMaxAssign = 512;
constexpr int kMlMaxExperts = 1024;
constexpr int64_t kMlMaxStride = 1 << 23;  // of x: 32-bit offsets over 64 rows
constexpr int kMlMaxSplits = 16;
constexpr int64_t kMlMaxSize = 1 << 18;    // of H and I: grids under 2^32 threads
constexpr int kMlTokenLds = 128 << 10;      // a group's tokens, 4-bit weights
constexpr int kMlMaxHiddenW4 = kMlTokenLds / 8;  // ... of four rows
constexpr int kUpWaves = 4, kDownWaves = 8;      // 16-bit weights
constexpr int kUpWavesW4 = 8, kShareWavesW4 = 4, kDownWavesW4 = 4;  // 4-bit weights
constexpr int kDownSlabsW4 = 2;                  // slabs of 16 columns a wave of theirs holds

struct MlArgs {
  const void* x;
  int64_t xs;
  const void* ids;
  int id_bytes;
  const void* weights;
  int weight_dtype;
  int N, top_k, A, E, H, I;
  WeightView w1, w2;
  void* act;          // [A][I]
  int* gexpert;       // [0]: number of groups, then each group's expert
  int16_t* glist;     // [group][16] assignments, -1: none
  float* part;        // the second kernel's partials
  uint32_t* counters; // one per slab set of the second kernel
  void* out;
  int64_t os;
  int tile;           // assignments of a group: 4, 8 or 16
  int max_groups;     // groups that the assignments can form
  int slabs;          // column slabs (second kernel: slab sets) of the grid
  int per_wg, wk;     // 4 bits, first kernel: slabs of a workgroup, waves that share a slab's k
  int splits;         // of the second kernel's work
  bool packed_out;    // out's rows are 8-byte aligned
  uint32_t* err;
};

__device__ __forceinline__ int64_t ml_id(const MlArgs& a, int i) {
  return a.id_bytes == 8 ? static_cast<const int64_t*>(a.ids)[i] : static_cast<const int32_t*>(a.ids)[i];
}

__device__ __forceinline__ int lanes_below(uint64_t mask, int lane) {
  return static_cast<int>(__popcll(mask & ((uint64_t(1) << lane) - 1)));
}

// The u-th group: its expert (-1: there are fewer) and, in the wave's list, its assignments. `lead`: the
// workgroup that reports for all; `record`: the one that leaves the group to the second kernel.
template <int W>
struct GroupLds {
  int count[kMlMaxExperts];
  int16_t expert[kMlMaxAssign];  // of each assignment, -1: none
  int list[W][kMlTile];
};

template <int W>
__device__ __forceinline__ int find_group(const MlArgs& a, int u, bool lead, bool record, GroupLds<W>& g) {
  const int lane = threadIdx.x & (kWave - 1);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  int* const list = g.list[wave];
  int expert = -1, groups = 0;
  bool bad = false;
  if (a.A <= kWave) {
    // An assignment a lane, no LDS and no barrier: every wave finds the group by itself, in the order of
    // the experts' first assignments.
    const int64_t id = lane < a.A ? ml_id(a, lane) : -1;
    const int e = id >= 0 && id < a.E ? static_cast<int>(id) : -1;
    bad = e < 0 && id != -1;
    int before = 0;  // earlier assignments of this one's expert
    for (int j = 0; j < a.A; ++j) before += __builtin_amdgcn_readlane(e, j) == e && j < lane ? 1 : 0;
    const uint64_t leads = __ballot(e >= 0 && before % a.tile == 0);
    groups = static_cast<int>(__popcll(leads));
    if (u < groups) {
      const uint64_t me = __ballot((leads >> lane & 1) != 0 && lanes_below(leads, lane) == u);
      const int l = static_cast<int>(__ffsll(static_cast<unsigned long long>(me))) - 1;
      expert = __builtin_amdgcn_readlane(e, l);
      const int at = before - __builtin_amdgcn_readlane(before, l);
      if (lane < kMlTile) list[lane] = -1;
      asm volatile("" ::: "memory");
      if (e == expert && at >= 0 && at < a.tile) list[at] = lane;
      asm volatile("" ::: "memory");
    }
  } else {
    for (int e = threadIdx.x; e < a.E; e += blockDim.x) g.count[e] = 0;
    __syncthreads();
    for (int i = threadIdx.x; i < a.A; i += blockDim.x) {
      const int64_t e = ml_id(a, i);
      const bool ok = e >= 0 && e < a.E;
      if (ok) atomicAdd(&g.count[e], 1);
      else bad |= e != -1;
      g.expert[i] = ok ? static_cast<int16_t>(e) : static_cast<int16_t>(-1);
    }
    __syncthreads();
    int rank = 0;  // every wave finds the same
    for (int e0 = 0; e0 < a.E; e0 += kWave) {
      const int n = e0 + lane < a.E ? (g.count[e0 + lane] + a.tile - 1) / a.tile : 0;
      int upto = n;  // inclusive prefix over lanes
#pragma unroll
      for (int s = 1; s < kWave; s *= 2) {
        const int v = __shfl_up(upto, s);
        if (lane >= s) upto += v;
      }
      const uint64_t past = __ballot(groups + upto > u);
      if (past != 0 && expert < 0) {
        const int l = static_cast<int>(__ffsll(static_cast<unsigned long long>(past))) - 1;
        expert = e0 + l;
        rank = (u - groups - (__shfl(upto, l) - __shfl(n, l))) * a.tile;
      }
      groups += __shfl(upto, kWave - 1);
    }
    if (expert >= 0) {
      if (lane < kMlTile) list[lane] = -1;
      asm volatile("" ::: "memory");
      int seen = 0;
      for (int i0 = 0; i0 < a.A; i0 += kWave) {
        const bool mine = i0 + lane < a.A && g.expert[i0 + lane] == expert;
        const uint64_t m = __ballot(mine);
        const int at = seen + lanes_below(m, lane) - rank;
        if (mine && at >= 0 && at < a.tile) list[at] = i0 + lane;
        seen += static_cast<int>(__popcll(m));
      }
      asm volatile("" ::: "memory");
    }
  }
  if (lead && bad) atomicOr(a.err, EMBER_ERR_EXPERT_ID);
  if (lead && threadIdx.x == 0) a.gexpert[0] = groups;
  expert = __builtin_amdgcn_readfirstlane(expert);
  if (expert >= 0 && record && threadIdx.x < kMlTile) {
    a.glist[u * kMlTile + threadIdx.x] = static_cast<int16_t>(list[threadIdx.x]);
    if (threadIdx.x == 0) a.gexpert[1 + u] = expert;
  }
  return expert;
}

template <typename T>
__global__ void __launch_bounds__(kUpWaves * kWave)
k_moe_layer_up(MlArgs a) {
  __shared__ GroupLds<kUpWaves> group;
  __shared__ __attribute__((aligned(16))) f32x4 red[kUpWaves][2][kWave];
  const int lane = threadIdx.x & (kWave - 1);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int u = blockIdx.x / a.slabs;
  const int slab = blockIdx.x - u * a.slabs;
  const int expert = find_group<kUpWaves>(a, u, blockIdx.x == 0, slab == 0, group);
  if (expert < 0) return;
  const int* list = group.list[wave];
  const int lead = list[0], slot = list[lane & 15];  // a row past the group's end repeats its first
  const T* xrow = static_cast<const T*>(a.x) + static_cast<int64_t>((slot >= 0 ? slot : lead) / a.top_k) * a.xs +
                  8 * (lane >> 4);
  const T* wp[2] = {half_slab<T>(a.w1, expert, slab, 0, lane), half_slab<T>(a.w1, expert, slab, 1, lane)};
  const int nb = a.w1.nb;
  f32x4 acc[1][2] = {{f32x4{0.f, 0.f, 0.f, 0.f}, f32x4{0.f, 0.f, 0.f, 0.f}}};
  using S = HalfStage<T, 2>;
  stream<S, 4>(
      0, wave < nb ? (nb - wave + kUpWaves - 1) / kUpWaves : 0,
      [&](S& st, int j) {
        const int b = min(wave + j * kUpWaves, nb - 1);
#pragma unroll
        for (int r = 0; r < 2; ++r) st.load(r, wp[r], b, a.w1.bs, a.w1.hs);
        st.load_x(xrow, b);
      },
      [&](const S& st, int) { st.compute(acc); });
  red[wave][0][lane] = acc[0][0];
  red[wave][1][lane] = acc[0][1];
  __syncthreads();
  // wave i finishes slots 4 (l / 16) + i
  float g = 0.f, up = 0.f;
#pragma unroll
  for (int q = 0; q < kUpWaves; ++q) {
    g += red[q][0][lane][wave];
    up += red[q][1][lane][wave];
  }
  const int id = list[4 * (lane >> 4) + wave];
  if (id >= 0)
    static_cast<T*>(a.act)[static_cast<int64_t>(id) * a.I + slab * 16 + (lane & 15)] = from_f32<T>(silu_mul(g, up));
}

// 4-bit experts, groups of 4 XI assignments. The group's tokens are put into LDS once; then each wave
// streams whole slabs by itself (wk = 1), or the waves share one slab's k (few groups).
template <typename T, int GPB, int XI>
__global__ void __launch_bounds__(kUpWavesW4 * kWave)
k_moe_layer_up_w4(MlArgs a) {
  using X = XBlock<1, XI>;
  __shared__ GroupLds<kUpWavesW4> group;
  extern __shared__ __attribute__((aligned(16))) u32x4 tokens[];  // [block][64 XI], then the waves' sums
  const int lane = threadIdx.x & (kWave - 1);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int sets = (a.slabs + a.per_wg - 1) / a.per_wg;
  const int u = blockIdx.x / sets;
  const int first = (blockIdx.x - u * sets) * a.per_wg;
  const int expert = find_group<kUpWavesW4>(a, u, blockIdx.x == 0, first == 0, group);
  if (expert < 0) return;
  const int* list = group.list[wave];
  const int nb = a.w1.nb;
  const int64_t slab_bytes = w4_slab_bytes(nb, GPB);
  const uint8_t* w = static_cast<const uint8_t*>(a.w1.w) + expert * a.w1.es;

  // item j of this wave: block b of slab s, both in steps
  const int s0 = a.wk == 1 ? first + wave : first, s_step = a.wk == 1 ? kUpWavesW4 : 1;
  const int b0 = a.wk == 1 ? 0 : wave, b_step = a.wk;
  const int s_end = min(first + a.per_wg, a.slabs);
  const int slabs = s0 < s_end ? (s_end - s0 + s_step - 1) / s_step : 0;
  const int blocks = b0 < nb ? (nb - b0 + b_step - 1) / b_step : 0;
  struct Cursor {
    int s, j;
  };
  Cursor ld{0, 0}, cs{0, 0};
  f32x4 acc[1][2] = {{f32x4{0.f, 0.f, 0.f, 0.f}, f32x4{0.f, 0.f, 0.f, 0.f}}};
  auto finish = [&](int slab, f32x4 g, f32x4 up) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int id = list[4 * (lane >> 4) + i];
      if (id >= 0)
        static_cast<T*>(a.act)[static_cast<int64_t>(id) * a.I + slab * 16 + (lane & 15)] =
            from_f32<T>(silu_mul(g[i], up[i]));
    }
  };
  using B = W4Block<2, GPB>;
  bool staged = false;
  auto stage = [&]() {  // the tokens into LDS, once the first weights are on their way
    staged = true;
    int off[XI];
    const BufferRsrc xr = buffer(a.x, static_cast<int>(((a.N - 1) * a.xs + a.H) * 2));
#pragma unroll
    for (int i = 0; i < XI; ++i) {
      const int id = list[4 * i + (lane >> 4)];
      off[i] = (id >= 0 ? id : list[0]) / a.top_k * static_cast<int>(a.xs) * 2 + 16 * (lane & 15);
    }
    for (int b = wave; b < nb; b += static_cast<int>(blockDim.x) / kWave) {
      X x;
      x.load(xr, off, b, a.H, lane);
      x.put(tokens + b * X::kPieces, lane);
    }
    __syncthreads();
  };
  stream<B, 4>(
      0, slabs * blocks,
      [&](B& st, int) {
        const int s = s0 + min(ld.s, slabs - 1) * s_step;
        const int b = b0 + ld.j * b_step;
        const uint8_t* at = w + 2 * s * slab_bytes;
#pragma unroll
        for (int r = 0; r < 2; ++r) st.load(r, buffer(at + r * slab_bytes, static_cast<int>(slab_bytes)), b, nb, lane);
        if (++ld.j == blocks) {
          ld.j = 0;
          ++ld.s;
        }
      },
      [&](const B& st, int) {
        if (!staged) stage();
        const u32x4* mine = tokens + (b0 + cs.j * b_step) * X::kPieces;
        st.template compute<T, 1>([&](int, int f) { return X::frag(mine, 0, f, lane); }, acc);
        if (++cs.j == blocks) {
          if (a.wk == 1) {
            finish(s0 + cs.s * s_step, acc[0][0], acc[0][1]);
            acc[0][0] = acc[0][1] = f32x4{0.f, 0.f, 0.f, 0.f};
          }
          cs.j = 0;
          ++cs.s;
        }
      });
  if (!staged) stage();  // a wave without work: the others wait for its share of the tokens
  if (a.wk == 1) return;
  f32x4* const red = reinterpret_cast<f32x4*>(tokens + nb * X::kPieces);
  red[(wave * 2) * kWave + lane] = acc[0][0];
  red[(wave * 2 + 1) * kWave + lane] = acc[0][1];
  __syncthreads();
  if (wave != 0) return;
  f32x4 g = red[lane], up = red[kWave + lane];
  for (int q = 1; q < a.wk; ++q) {
    g += red[2 * q * kWave + lane];
    up += red[(2 * q + 1) * kWave + lane];
  }
  finish(first, g, up);
}

// The second kernel: what its two forms share. R slabs of 16 columns a workgroup, W waves.
template <typename T, int R, int W>
struct Down {
  static constexpr int kCols = 16 * R;
  const MlArgs& a;
  int lane, wave, split, set, G;
  float *all, *sums, *wts;
  int16_t *lists, *experts;

  __device__ __forceinline__ Down(const MlArgs& args, float* lds) : a(args) {
    lane = threadIdx.x & (kWave - 1);
    wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    split = blockIdx.x / a.slabs;
    set = blockIdx.x - split * a.slabs;
    G = __builtin_amdgcn_readfirstlane(a.gexpert[0]);
    all = lds;  // [wave][N][kCols]
    sums = all + wave * a.N * kCols;
    wts = all + W * a.N * kCols;
    lists = reinterpret_cast<int16_t*>(wts + (a.A + 3) / 4 * 4);
    experts = lists + a.max_groups * kMlTile;  // all that there can be: their loads need not wait for G
    for (int i = lane; i < a.N * kCols; i += kWave) sums[i] = 0.f;
    for (int i = threadIdx.x; i < a.A; i += W * kWave) {
      float w;
      if (a.weight_dtype == EMBER_F32) w = static_cast<const float*>(a.weights)[i];
      else if (a.weight_dtype == EMBER_F16) w = to_f32(static_cast<const _Float16*>(a.weights)[i]);
      else w = to_f32(static_cast<const __bf16*>(a.weights)[i]);
      wts[i] = w;
    }
    for (int i = threadIdx.x; i < a.max_groups * kMlTile / 8; i += W * kWave)
      reinterpret_cast<u32x4*>(lists)[i] = reinterpret_cast<const u32x4*>(a.glist)[i];
    for (int i = threadIdx.x; i < a.max_groups; i += W * kWave) experts[i] = static_cast<int16_t>(a.gexpert[1 + i]);
    __syncthreads();
  }
  // this wave's items, of n a group
  __device__ __forceinline__ int item(int n, int end) const {
    return static_cast<int>(static_cast<int64_t>(G) * n * (split * W + wave + end) / (a.splits * W));
  }
  __device__ __forceinline__ int expert(int u) const {
    return __builtin_amdgcn_readfirstlane(static_cast<int>(experts[u]));
  }
  // a row past the group's end repeats its first
  __device__ __forceinline__ int assignment(int u, int i) const {
    const int id = lists[u * kMlTile + i];
    return id >= 0 ? id : static_cast<int>(lists[u * kMlTile]);
  }
  // the end of this wave's share of group u: weight it and add it to the tokens' sums
  __device__ __forceinline__ void flush(int u, f32x4 (&acc)[1][R]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int id = lists[u * kMlTile + 4 * (lane >> 4) + i];
      if (id >= 0) {
        // atomics, because a token may name one expert twice; the wave's own array
#pragma unroll
        for (int r = 0; r < R; ++r)
          __hip_atomic_fetch_add(&sums[id / a.top_k * kCols + 16 * r + (lane & 15)], wts[id] * acc[0][r][i],
                                 __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
      }
    }
#pragma unroll
    for (int r = 0; r < R; ++r) acc[0][r] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  // The waves' sums in order, then the splits': by the last to arrive, in their order. Four columns a
  // thread; the partials are [set][split][N][kCols].
  __device__ __forceinline__ void join(int* last) {
    __syncthreads();
    const int n4 = a.N * kCols / 4;
    auto emit = [&](int i, f32x4 y) {
      Pack<T, 4> o;
#pragma unroll
      for (int c = 0; c < 4; ++c) o.v[c] = from_f32<T>(y[c]);
      T* p = static_cast<T*>(a.out) + static_cast<int64_t>(4 * i / kCols) * a.os + set * kCols + 4 * i % kCols;
      if (a.packed_out) store_pack<T, 4>(p, o);
      else
        for (int c = 0; c < 4; ++c) p[c] = o.v[c];
    };
    const CoherentRsrc rs = coherent_rsrc(a.part + static_cast<int64_t>(set) * a.splits * a.N * kCols, a.splits * a.N * kCols);
    for (int i = threadIdx.x; i < n4; i += W * kWave) {
      f32x4 y = reinterpret_cast<const f32x4*>(all)[i];
#pragma unroll
      for (int w = 1; w < W; ++w) y += reinterpret_cast<const f32x4*>(all)[w * n4 + i];
      if (a.splits == 1) emit(i, y);
      else store_coherent<4>(rs, (split * n4 + i) * 16, y);
    }
    if (a.splits == 1) return;
    __builtin_amdgcn_s_waitcnt(0);
    __syncthreads();
    if (threadIdx.x == 0) {
      const uint32_t prev = __hip_atomic_fetch_add(a.counters + set, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      *last = prev == static_cast<uint32_t>(a.splits) - 1;
      if (*last) __hip_atomic_store(a.counters + set, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    __syncthreads();
    if (!*last) return;
    constexpr int B = 8;  // loads in flight
    for (int i = threadIdx.x; i < n4; i += W * kWave) {
      f32x4 y = {0.f, 0.f, 0.f, 0.f};
      for (int s0 = 0; s0 < a.splits; s0 += B) {
        f32x4 v[B];
#pragma unroll
        for (int s = 0; s < B; ++s) v[s] = load_coherent<4>(rs, (min(s0 + s, a.splits - 1) * n4 + i) * 16);
#pragma unroll
        for (int s = 0; s < B; ++s) y += s0 + s < a.splits ? v[s] : f32x4{0.f, 0.f, 0.f, 0.f};
      }
      emit(i, y);
    }
  }
};

template <typename T>
__global__ void __launch_bounds__(kDownWaves * kWave)
k_moe_layer_down(MlArgs a) {
  extern __shared__ __attribute__((aligned(16))) float lds[];
  __shared__ int last;
  Down<T, 1, kDownWaves> d(a, lds);
  const int nb = a.w2.nb, i0 = d.item(nb, 0), i1 = d.item(nb, 1);
  f32x4 acc[1][1] = {{f32x4{0.f, 0.f, 0.f, 0.f}}};
  int lu = -1;  // the group whose pointers the loads use
  const T* act = static_cast<const T*>(a.act) + 8 * (d.lane >> 4);
  const T* xrow = act;
  const T* wp = nullptr;
  using S = HalfStage<T, 1>;
  stream<S, 4>(
      i0, i1,
      [&](S& st, int item) {
        const int it = min(item, i1 - 1);
        const int u = it / nb, b = it - u * nb;
        if (u != lu) {  // uniform
          lu = u;
          xrow = act + static_cast<int64_t>(d.assignment(u, d.lane & 15)) * a.I;
          wp = half_slab<T>(a.w2, d.expert(u), d.set, 0, d.lane);
        }
        st.load(0, wp, b, a.w2.bs, a.w2.hs);
        st.load_x(xrow, b);
      },
      [&](const S& st, int item) {
        st.compute(acc);
        const int u = item / nb;
        if (item - u * nb == nb - 1 || item == i1 - 1) d.flush(u, acc);  // uniform
      });
  d.join(&last);
}

template <typename T, int GPB, int XI>
__global__ void __launch_bounds__(kDownWavesW4 * kWave, 4)
k_moe_layer_down_w4(MlArgs a) {
  using X = XBlock<1, XI>;
  constexpr int R = kDownSlabsW4;
  extern __shared__ __attribute__((aligned(16))) float lds[];
  __shared__ u32x4 rows[kDownWavesW4][X::kPieces];
  __shared__ int last;
  Down<T, R, kDownWavesW4> d(a, lds);
  const int nb = a.w2.nb, i0 = d.item(nb, 0), i1 = d.item(nb, 1);
  const int64_t slab_bytes = w4_slab_bytes(nb, GPB);
  const BufferRsrc ar = buffer(a.act, a.A * a.I * 2);
  f32x4 acc[1][R];
#pragma unroll
  for (int r = 0; r < R; ++r) acc[0][r] = f32x4{0.f, 0.f, 0.f, 0.f};
  struct Stage {
    W4Block<R, GPB> w;
    X x;
  };
  int lu = -1;  // the group whose rows and weights the loads use
  int off[XI];
#pragma unroll
  for (int i = 0; i < XI; ++i) off[i] = 0;
  const uint8_t* w = nullptr;
  stream<Stage, XI == 1 ? 4 : (XI == 2 ? 3 : 2)>(
      i0, i1,
      [&](Stage& st, int item) {
        const int it = min(item, i1 - 1);
        const int u = it / nb, b = it - u * nb;
        if (u != lu) {  // uniform
          lu = u;
#pragma unroll
          for (int i = 0; i < XI; ++i)
            off[i] = d.assignment(u, 4 * i + (d.lane >> 4)) * a.I * 2 + 16 * (d.lane & 15);
          w = static_cast<const uint8_t*>(a.w2.w) + d.expert(u) * a.w2.es + d.set * R * slab_bytes;
        }
#pragma unroll
        for (int r = 0; r < R; ++r)
          st.w.load(r, buffer(w + r * slab_bytes, static_cast<int>(slab_bytes)), b, nb, d.lane);
        st.x.load(ar, off, b, a.I, d.lane);
      },
      [&](const Stage& st, int item) {
        st.x.put(rows[d.wave], d.lane);
        st.w.template compute<T, 1>([&](int, int f) { return X::frag(rows[d.wave], 0, f, d.lane); }, acc);
        const int u = item / nb;
        if (item - u * nb == nb - 1 || item == i1 - 1) d.flush(u, acc);  // uniform
      });
  d.join(&last);
}

// Assignments of a group: 16 rows are one MFMA tile; 4-bit weights stream fast enough that 16 rows of
// tokens in LDS would cost them occupancy, so their groups are as small as holds nearly every expert's
// share of a mean of 2.5 and of 5, and take at most kMlTokenLds bytes.
int group_tile(int64_t A, int64_t E, int64_t H, bool w4) {
  if (!w4) return kMlTile;
  int tile = 2 * A <= 5 * E ? 4 : (A <= 5 * E ? 8 : 16);
  while (tile * cdiv(H, kW4Block) * kW4Block * 2 > kMlTokenLds) tile /= 2;
  return tile;
}

// Groups that A assignments to E experts can form.
int64_t max_groups(int64_t A, int64_t E, int tile) { return std::min(A, std::min(A, E) + A / tile); }

// Splits of the second kernel's work: 16 waves a CU, as long as each of them gets two blocks of k where
// every routed expert has one group.
int64_t down_splits(int64_t A, int64_t E, int64_t sets, int64_t blocks, int waves) {
  const int64_t cus = std::max(1, device_cu_count());
  const int64_t want = std::max<int64_t>(1, (16 / waves * cus + sets / 2) / sets);
  const int64_t most = std::max<int64_t>(1, std::min(A, E) * blocks / (2 * waves));
  return std::min<int64_t>(kMlMaxSplits, std::min(want, most));
}

struct MlLayout {
  int64_t act, gexpert, glist, part, partial, counters;  // offsets, end of the partials, bytes of counters
};

// The same for 16 and 4 bits, at the larger's needs.
MlLayout ml_layout(int64_t N, int64_t top_k, int64_t E, int64_t H, int64_t I) {
  const int64_t A = N * top_k, g = max_groups(A, E, 4);
  auto up = [](int64_t v) { return (v + 255) / 256 * 256; };
  MlLayout l;
  l.act = 0;
  l.gexpert = up(A * I * 2);
  l.glist = l.gexpert + up(4 * (g + 1));
  l.part = l.glist + up(2 * kMlTile * g);
  l.partial = l.part + up(kMlMaxSplits * N * H * 4);
  l.counters = up(H / 16 * 4);
  return l;
}

bool ml_sizes_ok(int64_t N, int64_t top_k, int64_t E, int64_t H, int64_t I) {
  return N >= 0 && N <= kMlMaxTokens && top_k >= 1 && N * top_k <= kMlMaxAssign && top_k <= kMlMaxAssign && E >= 1 &&
         E <= kMlMaxExperts && H >= 32 && I >= 32 && H % 32 == 0 && I % 32 == 0 && H <= kMlMaxSize && I <= kMlMaxSize;
}

size_t down_lds(const MlArgs& a, int waves, int cols) {
  return 4 * (size_t(waves) * a.N * cols + a.A + 3) + 2 * size_t(a.max_groups) * (kMlTile + 1) + 16;
}

template <typename T>
int ml_half(MlArgs a, hipStream_t s) {
  a.slabs = a.I / 16;
  const int64_t grid = static_cast<int64_t>(a.max_groups) * a.slabs;
  k_moe_layer_up<T><<<dim3(static_cast<unsigned>(grid)), kUpWaves * kWave, 0, s>>>(a);
  if (const int st = launch_status(); st != EMBER_OK) return st;
  a.slabs = a.H / 16;
  a.splits = static_cast<int>(down_splits(a.A, a.E, a.slabs, a.w2.nb, kDownWaves));
  k_moe_layer_down<T><<<dim3(static_cast<unsigned>(a.slabs * a.splits)), kDownWaves * kWave,
                        down_lds(a, kDownWaves, 16), s>>>(a);
  return launch_status();
}

template <typename T, int GPB, int XI>
int ml_up_w4(MlArgs a, hipStream_t s) {
  a.slabs = a.I / 16;
  const int64_t groups = a.max_groups, cus = std::max(1, device_cu_count());
  // Whole slabs a wave once they fill the chip twice over; until then the waves share a slab's k: four of
  // them, so that a token's workgroups are on the chip at once (Moonlight's 528: 8 waves each took two turns)
  const bool whole = groups * a.slabs >= 2 * kUpWavesW4 * cus;
  const int waves = whole ? kUpWavesW4 : kShareWavesW4;
  a.wk = whole ? 1 : waves;
  a.per_wg = whole ? waves : 1;
  const size_t lds = 16 * (size_t(a.w1.nb) * XBlock<1, XI>::kPieces + (whole ? 0 : waves * 2 * kWave));
  auto kernel = k_moe_layer_up_w4<T, GPB, XI>;
  if (lds > 65536 - sizeof(GroupLds<kUpWavesW4>) &&
      hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize,
                          static_cast<int>(lds)) != hipSuccess)
    return EMBER_ENODEV;
  kernel<<<dim3(static_cast<unsigned>(groups * cdiv(a.slabs, a.per_wg))), waves * kWave, lds, s>>>(a);
  return launch_status();
}

template <typename T, int GPB, int XI>
int ml_down_w4(MlArgs a, hipStream_t s) {
  a.slabs = a.H / (16 * kDownSlabsW4);
  a.splits = static_cast<int>(down_splits(a.A, a.E, a.slabs, a.w2.nb, kDownWavesW4));
  k_moe_layer_down_w4<T, GPB, XI><<<dim3(static_cast<unsigned>(a.slabs * a.splits)), kDownWavesW4 * kWave,
                                    down_lds(a, kDownWavesW4, 16 * kDownSlabsW4), s>>>(a);
  return launch_status();
}

template <typename T, int XI>
int ml_w4(const MlArgs& a, int gpb1, int gpb2, hipStream_t s) {
  const int st = gpb1 == 1 ? ml_up_w4<T, 1, XI>(a, s) : (gpb1 == 2 ? ml_up_w4<T, 2, XI>(a, s) : ml_up_w4<T, 4, XI>(a, s));
  if (st != EMBER_OK) return st;
  return gpb2 == 1 ? ml_down_w4<T, 1, XI>(a, s) : (gpb2 == 2 ? ml_down_w4<T, 2, XI>(a, s) : ml_down_w4<T, 4, XI>(a, s));
}

template <typename T>
int ml_run(const MlArgs& a, int gpb1, int gpb2, hipStream_t s) {
  if (gpb1 == 0) return ml_half<T>(a, s);
  return a.tile == 4 ? ml_w4<T, 1>(a, gpb1, gpb2, s)
                     : (a.tile == 8 ? ml_w4<T, 2>(a, gpb1, gpb2, s) : ml_w4<T, 4>(a, gpb1, gpb2, s));
}

struct MlCall {
  const void* x;
  int64_t xs;
  const void* ids;
  int id_bytes;
  const void* weights;
  int weight_dtype, dtype;
  int64_t N, top_k, E, H, I;
  void* workspace;
  int64_t workspace_bytes;
  void* out;
  int64_t os;
  void* stream;
};

// gpb1, gpb2: groups a block of the two 4-bit weights, 0 for 16 bits.
int ml_call(const MlCall& c, const WeightView& w1, const WeightView& w2, int gpb1, int gpb2) {
  if (!ml_sizes_ok(c.N, c.top_k, c.E, c.H, c.I) || (c.dtype != EMBER_F16 && c.dtype != EMBER_BF16) ||
      (c.id_bytes != 4 && c.id_bytes != 8) || dtype_size(c.weight_dtype) == 0 || c.xs < 0 || c.xs > kMlMaxStride ||
      c.os < 0)
    return EMBER_EINVAL;
  if (c.N == 0) return EMBER_OK;
  const MlLayout l = ml_layout(c.N, c.top_k, c.E, c.H, c.I);
  if (c.x == nullptr || c.ids == nullptr || c.weights == nullptr || w1.w == nullptr || w2.w == nullptr ||
      c.out == nullptr || c.workspace == nullptr || c.workspace_bytes < l.partial + l.counters)
    return EMBER_EINVAL;
  if (!aligned16(c.x) || c.xs % 8 != 0 || !aligned16(w1.w) || !aligned16(w2.w) || !aligned16(c.workspace) ||
      c.workspace_bytes % 16 != 0)
    return EMBER_EALIGN;
  uint32_t* err = device_error_word();
  if (err == nullptr) return EMBER_ENODEV;
  uint8_t* ws = static_cast<uint8_t*>(c.workspace);
  MlArgs a{};
  a.x = c.x;
  a.xs = c.xs;
  a.ids = c.ids;
  a.id_bytes = c.id_bytes;
  a.weights = c.weights;
  a.weight_dtype = c.weight_dtype;
  a.N = static_cast<int>(c.N);
  a.top_k = static_cast<int>(c.top_k);
  a.A = static_cast<int>(c.N * c.top_k);
  a.E = static_cast<int>(c.E);
  a.H = static_cast<int>(c.H);
  a.I = static_cast<int>(c.I);
  a.w1 = w1;
  a.w2 = w2;
  a.act = ws + l.act;
  a.gexpert = reinterpret_cast<int*>(ws + l.gexpert);
  a.glist = reinterpret_cast<int16_t*>(ws + l.glist);
  a.part = reinterpret_cast<float*>(ws + l.part);
  a.counters = reinterpret_cast<uint32_t*>(ws + c.workspace_bytes - l.counters);
  a.out = c.out;
  a.os = c.os;
  a.packed_out = (reinterpret_cast<uintptr_t>(c.out) | (c.os * 2)) % 8 == 0;
  a.tile = group_tile(a.A, a.E, a.H, gpb1 > 0);
  a.max_groups = static_cast<int>(max_groups(a.A, a.E, a.tile));
  a.err = err;
  hipStream_t s = static_cast<hipStream_t>(c.stream);
  return c.dtype == EMBER_F16 ? ml_run<_Float16>(a, gpb1, gpb2, s) : ml_run<__bf16>(a, gpb1, gpb2, s);
}

constexpr int64_t kUnit = 8192;  // elements of ember_moe_gate_up_silu_pack_weight's unit

WeightView rows_view(const void* w, int64_t expert_stride, int64_t row_stride, int64_t part_rows, int64_t k) {
  WeightView v{};
  v.w = w;
  v.es = expert_stride;
  v.s4 = 64 * row_stride;
  v.s1 = 16 * row_stride;
  v.ps = part_rows * row_stride;
  v.bs = 64;
  v.hs = 32;
  v.lr = row_stride;
  v.lg = 8;
  v.nb = static_cast<int>(k / 64);
  return v;
}

// The packed down weight: [expert][row / 16][k / 32][lane][8], one contiguous stream per slab.
struct DownPackArgs {
  const void* w;
  int64_t es, rs;
  uint8_t* dst;
  int rows, k;
  int64_t pieces;
};

__global__ void __launch_bounds__(256) k_moe_down_pack(DownPackArgs a) {
  const int steps = a.k / 32, slabs = a.rows / 16;
  for (int64_t t = int64_t(blockIdx.x) * 256 + threadIdx.x; t < a.pieces; t += int64_t(gridDim.x) * 256) {
    const int lane = static_cast<int>(t & 63);
    int64_t q = t >> 6;
    const int step = static_cast<int>(q % steps);
    q /= steps;
    const int64_t e = q / slabs, slab = q % slabs;
    const int64_t at = e * a.es + (16 * slab + (lane & 15)) * a.rs + 32 * step + 8 * (lane >> 4);
    reinterpret_cast<u32x4*>(a.dst)[t] = *reinterpret_cast<const u32x4*>(static_cast<const uint16_t*>(a.w) + at);
  }
}

}  // namespace
}  // namespace ember

using namespace ember;

extern "C" {

int64_t ember_moe_layer_workspace_bytes(int64_t num_tokens, int64_t top_k, int64_t num_experts, int64_t hidden,
                                        int64_t inter, int64_t* counter_bytes) {
  if (!ml_sizes_ok(num_tokens, top_k, num_experts, hidden, inter)) return -1;
  const MlLayout l = ml_layout(num_tokens, top_k, num_experts, hidden, inter);
  if (counter_bytes != nullptr) *counter_bytes = l.counters;
  return l.partial + l.counters;
}

int ember_moe_layer(const void* x, int64_t x_row_stride, const void* topk_ids, int id_bytes, const void* topk_weights,
                    int weight_dtype, int64_t num_tokens, int64_t top_k, const void* w_gate_up,
                    int64_t gate_up_expert_stride, int64_t gate_up_row_stride, const void* w_down,
                    int64_t down_expert_stride, int64_t down_row_stride, int dtype, int64_t num_experts, int64_t hidden,
                    int64_t inter, void* workspace, int64_t workspace_bytes, void* out, int64_t out_row_stride,
                    void* stream) {
  if (hidden % 64 != 0 || inter % 64 != 0) return EMBER_EINVAL;
  if ((gate_up_row_stride | gate_up_expert_stride | down_row_stride | down_expert_stride) % 8 != 0) return EMBER_EALIGN;
  WeightView w1, w2;
  if (gate_up_row_stride != 0) {
    w1 = rows_view(w_gate_up, gate_up_expert_stride, gate_up_row_stride, inter, hidden);
  } else {  // ember_moe_gate_up_silu_pack_weight's units
    w1 = WeightView{w_gate_up, 2 * inter * hidden, kUnit, 1024, 512, inter / 64 * kUnit, 4096, 8, 128,
                    static_cast<int>(hidden / 64)};
  }
  if (down_row_stride != 0) {
    w2 = rows_view(w_down, down_expert_stride, down_row_stride, 0, inter);
  } else {  // ember_moe_down_pack_weight's slabs
    const int64_t slab = 16 * inter;
    w2 = WeightView{w_down, hidden * inter, 4 * slab, slab, 0, 1024, 512, 8, 128, static_cast<int>(inter / 64)};
  }
  return ml_call({x, x_row_stride, topk_ids, id_bytes, topk_weights, weight_dtype, dtype, num_tokens, top_k, num_experts,
                  hidden, inter, workspace, workspace_bytes, out, out_row_stride, stream},
                 w1, w2, 0, 0);
}

int ember_moe_layer_w4(const void* x, int64_t x_row_stride, const void* topk_ids, int id_bytes,
                       const void* topk_weights, int weight_dtype, int64_t num_tokens, int64_t top_k,
                       const void* packed_gate_up, int64_t gate_up_group, const void* packed_down, int64_t down_group,
                       int dtype, int64_t num_experts, int64_t hidden, int64_t inter, void* workspace,
                       int64_t workspace_bytes, void* out, int64_t out_row_stride, void* stream) {
  const int64_t b1 = ember_w4_packed_bytes(inter, hidden, gate_up_group, 1);
  const int64_t b2 = ember_w4_packed_bytes(hidden, inter, down_group, 0);
  if (b1 < 0 || b2 < 0 || hidden > kMlMaxHiddenW4) return EMBER_EINVAL;
  WeightView w1{}, w2{};
  w1.w = packed_gate_up;
  w1.es = b1;
  w1.nb = static_cast<int>(cdiv(hidden, kW4Block));
  w2.w = packed_down;
  w2.es = b2;
  w2.nb = static_cast<int>(cdiv(inter, kW4Block));
  return ml_call({x, x_row_stride, topk_ids, id_bytes, topk_weights, weight_dtype, dtype, num_tokens, top_k, num_experts,
                  hidden, inter, workspace, workspace_bytes, out, out_row_stride, stream},
                 w1, w2, w4_gpb(gate_up_group), w4_gpb(down_group));
}

int ember_moe_down_pack_weight(const void* w, int64_t w_expert_stride, int64_t w_row_stride, int dtype,
                               int64_t num_experts, int64_t hidden, int64_t inter, void* packed, void* stream) {
  if (w == nullptr || packed == nullptr || (dtype != EMBER_F16 && dtype != EMBER_BF16) || num_experts < 1 ||
      hidden < 16 || hidden % 16 != 0 || inter < 64 || inter % 64 != 0 || hidden > (1 << 24) || inter > (1 << 24))
    return EMBER_EINVAL;
  if (!aligned16(w) || !aligned16(packed) || w_expert_stride % 8 != 0 || w_row_stride % 8 != 0) return EMBER_EALIGN;
  DownPackArgs a{w, w_expert_stride, w_row_stride, static_cast<uint8_t*>(packed), static_cast<int>(hidden),
                 static_cast<int>(inter), num_experts * hidden * inter / 8};
  const int64_t grid = std::min<int64_t>(cdiv(a.pieces, 256), 65536);
  k_moe_down_pack<<<dim3(static_cast<unsigned>(grid)), 256, 0, static_cast<hipStream_t>(stream)>>>(a);
  return launch_status();
}

}  // extern "C"
