// The routed experts' whole layer for a decode step's tokens, in two kernels:
//   act[a, j] = round(silu(x[t] . W1[e, j]) * (x[t] . W1[e, I + j]))     a = t * top_k + c, e = ids[t, c]
//   out[t, n] = round(sum_c weights[t, c] * (W2[e, n] . act[a]))
// (fused_moe_forward, emberserve/model/moe_triton.py:332-345), over fp16/bf16 experts, unpacked or
// packed, and over 4-bit experts. g, u and the routed sum stay in fp32; act is rounded once, to be an
// MFMA operand.
//
// What bounds it: the weights of the experts that the step's tokens reach, each read once. The
// assignments of an expert form groups of 16 (an MFMA tile). Every workgroup of the first kernel finds
// its group in the routing ids by itself, so there is no alignment launch: group u of the experts in
// ascending order, with at most min(A, E) + A / 16 of them for A assignments. Its four waves share the
// group's k for 16 gate and 16 up rows and meet in LDS.
//
// The second kernel's workgroups hold 16 output columns each for all groups (times a split of the work):
// the waves cut the (group, k block) items of their columns into equal runs, whatever expert they belong
// to, and add each group's finished tile, weighted, to their own fp32 sums [token][16] in LDS. The sums
// of the waves, then of the splits (the last to arrive), are added in order, so that results do not
// depend on which wave was first.
#include <algorithm>

#include "w4.h"

namespace ember {
namespace {

constexpr int kMlTile = 16;             // assignments a group
constexpr int kMlMaxTokens = 64;
constexpr int kMlMaxAssign = 512;
constexpr int kMlMaxExperts = 1024;
constexpr int kUpWaves = 4;
constexpr int kDownWaves = 8;
constexpr int kMlMaxSplits = 16;

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
  int* glist;         // [group][16] assignments, -1: none
  float* part;        // [split][N][H]
  uint32_t* counters; // [H / 16]
  void* out;
  int64_t os;
  int slabs, splits;  // first kernel: column slabs; second: column slabs and splits
  uint32_t* err;
};

__device__ __forceinline__ int64_t ml_id(const MlArgs& a, int i) {
  return a.id_bytes == 8 ? static_cast<const int64_t*>(a.ids)[i] : static_cast<const int32_t*>(a.ids)[i];
}

__device__ __forceinline__ int lanes_below(uint64_t mask, int lane) {
  return static_cast<int>(__popcll(mask & ((uint64_t(1) << lane) - 1)));
}

template <typename T, int GPB, int D>
__global__ void __launch_bounds__(kUpWaves * kWave)
k_moe_layer_up(MlArgs a) {
  using S = Stage<T, 2, 1, GPB>;
  __shared__ int count[kMlMaxExperts];
  __shared__ int list[kMlTile];
  __shared__ int found[2];  // the group's expert and its first rank
  __shared__ __attribute__((aligned(16))) f32x4 red[kUpWaves][2][kWave];
  const int lane = threadIdx.x & (kWave - 1);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int u = blockIdx.x / a.slabs;
  const int slab = blockIdx.x - u * a.slabs;

  // The u-th group. Every wave would find the same; the first does, for all.
  for (int e = threadIdx.x; e < a.E; e += kUpWaves * kWave) count[e] = 0;
  if (threadIdx.x < kMlTile) list[threadIdx.x] = -1;
  __syncthreads();
  for (int i = threadIdx.x; i < a.A; i += kUpWaves * kWave) {
    const int64_t e = ml_id(a, i);
    if (e >= 0 && e < a.E) atomicAdd(&count[e], 1);
    else if (e != -1 && blockIdx.x == 0) atomicOr(a.err, EMBER_ERR_EXPERT_ID);
  }
  __syncthreads();
  if (wave == 0) {
    int before = 0, expert = -1, rank = 0;
    for (int e0 = 0; e0 < a.E; e0 += kWave) {
      const int g = e0 + lane < a.E ? (count[e0 + lane] + kMlTile - 1) / kMlTile : 0;
      int upto = g;  // inclusive prefix over lanes
#pragma unroll
      for (int s = 1; s < kWave; s *= 2) {
        const int v = __shfl_up(upto, s);
        if (lane >= s) upto += v;
      }
      const uint64_t past = __ballot(before + upto > u);
      if (past != 0 && expert < 0) {
        const int l = static_cast<int>(__ffsll(static_cast<unsigned long long>(past))) - 1;
        expert = e0 + l;
        rank = (u - before - (__shfl(upto, l) - __shfl(g, l))) * kMlTile;
      }
      before += __shfl(upto, kWave - 1);
    }
    if (blockIdx.x == 0 && lane == 0) a.gexpert[0] = before;
    if (expert >= 0) {
      int seen = 0;
      for (int i0 = 0; i0 < a.A; i0 += kWave) {
        const bool mine = i0 + lane < a.A && ml_id(a, i0 + lane) == expert;
        const uint64_t m = __ballot(mine);
        const int at = seen + lanes_below(m, lane) - rank;
        if (mine && at >= 0 && at < kMlTile) list[at] = i0 + lane;
        seen += static_cast<int>(__popcll(m));
      }
    }
    if (lane == 0) found[0] = expert;
  }
  __syncthreads();
  const int expert = __builtin_amdgcn_readfirstlane(found[0]);
  if (expert < 0) return;  // fewer groups than the grid allows for
  if (slab == 0 && threadIdx.x < kMlTile) {
    a.glist[u * kMlTile + threadIdx.x] = list[threadIdx.x];
    if (threadIdx.x == 0) a.gexpert[1 + u] = expert;
  }

  const int mine = max(list[lane & 15], 0);  // a row past the group's end repeats a real one
  const int first = list[0];
  const T* xrow = static_cast<const T*>(a.x) + static_cast<int64_t>((list[lane & 15] >= 0 ? mine : first) / a.top_k) * a.xs +
                  8 * (lane >> 4);
  const uint8_t* base[2];
  WeightPtr<T, GPB> wp[2];
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    if constexpr (GPB > 0)
      base[r] = static_cast<const uint8_t*>(a.w1.w) + expert * a.w1.es +
                static_cast<int64_t>(2 * slab + r) * a.w1.nb * w4_block_bytes(GPB);
    else
      wp[r].set(a.w1, expert, slab, r, lane);
  }
  S ring[D];
  f32x4 acc[1][2] = {{f32x4{0.f, 0.f, 0.f, 0.f}, f32x4{0.f, 0.f, 0.f, 0.f}}};
  const int nb = a.w1.nb;
  const int nj = wave < nb ? (nb - wave + kUpWaves - 1) / kUpWaves : 0;
  auto issue = [&](S& st, int j) {
    const int b = min(wave + j * kUpWaves, nb - 1);
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      if constexpr (GPB > 0) st.load_w4(r, base[r], b, lane);
      else st.load_half(r, wp[r].p, b, a.w1.bs, a.w1.hs);
    }
    st.load_x(0, xrow, b, a.H);
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

template <typename T, int GPB, int D>
__global__ void __launch_bounds__(kDownWaves * kWave)
k_moe_layer_down(MlArgs a) {
  using S = Stage<T, 1, 1, GPB>;
  // [wave][N][16] sums, then the assignments' weights [A], then the groups' lists [group][16] and experts
  extern __shared__ __attribute__((aligned(16))) float lds[];
  __shared__ int last;
  const int lane = threadIdx.x & (kWave - 1);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int split = blockIdx.x / a.slabs;
  const int slab = blockIdx.x - split * a.slabs;
  const int G = __builtin_amdgcn_readfirstlane(a.gexpert[0]);
  float* const sums = lds + wave * a.N * 16;
  float* const wts = lds + kDownWaves * a.N * 16;
  int16_t* const lists = reinterpret_cast<int16_t*>(wts + a.A);
  int16_t* const experts = lists + G * kMlTile;
  for (int i = lane; i < a.N * 16; i += kWave) sums[i] = 0.f;
  for (int i = threadIdx.x; i < a.A; i += kDownWaves * kWave) {
    float w;
    if (a.weight_dtype == EMBER_F32) w = static_cast<const float*>(a.weights)[i];
    else if (a.weight_dtype == EMBER_F16) w = to_f32(static_cast<const _Float16*>(a.weights)[i]);
    else w = to_f32(static_cast<const __bf16*>(a.weights)[i]);
    wts[i] = w;
  }
  for (int i = threadIdx.x; i < G * kMlTile; i += kDownWaves * kWave) lists[i] = static_cast<int16_t>(a.glist[i]);
  for (int i = threadIdx.x; i < G; i += kDownWaves * kWave) experts[i] = static_cast<int16_t>(a.gexpert[1 + i]);
  __syncthreads();

  // this wave's items (group, k block) [i0, i1)
  const int nb = a.w2.nb;
  const int items = G * nb, parts = a.splits * kDownWaves, me = split * kDownWaves + wave;
  const int i0 = static_cast<int>(static_cast<int64_t>(items) * me / parts);
  const int i1 = static_cast<int>(static_cast<int64_t>(items) * (me + 1) / parts);
  const T* act = static_cast<const T*>(a.act) + 8 * (lane >> 4);

  int lu = -1;  // the group whose pointers the loads use
  const T* xrow = act;
  const uint8_t* base = nullptr;
  WeightPtr<T, GPB> wp{};
  auto issue = [&](S& st, int item) {
    const int it = min(item, i1 - 1);
    const int u = it / nb, b = it - u * nb;
    if (u != lu) {  // uniform
      lu = u;
      const int e = __builtin_amdgcn_readfirstlane(static_cast<int>(experts[u]));
      const int id = lists[u * kMlTile + (lane & 15)];
      xrow = act + static_cast<int64_t>(id >= 0 ? id : lists[u * kMlTile]) * a.I;
      if constexpr (GPB > 0)
        base = static_cast<const uint8_t*>(a.w2.w) + e * a.w2.es + static_cast<int64_t>(slab) * nb * w4_block_bytes(GPB);
      else
        wp.set(a.w2, e, slab, 0, lane);
    }
    if constexpr (GPB > 0) st.load_w4(0, base, b, lane);
    else st.load_half(0, wp.p, b, a.w2.bs, a.w2.hs);
    st.load_x(0, xrow, b, a.I);
  };
  f32x4 acc[1][1] = {{f32x4{0.f, 0.f, 0.f, 0.f}}};
  auto consume = [&](const S& st, int item) {
    st.compute(acc);
    const int u = item / nb;
    if (item - u * nb != nb - 1 && item != i1 - 1) return;  // uniform
    // the end of this wave's share of the group: weight it and add it to the tokens' sums
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int id = lists[u * kMlTile + 4 * (lane >> 4) + i];
      if (id >= 0) {
        // an atomic, because a token may name one expert twice; the wave's own array
        __hip_atomic_fetch_add(&sums[id / a.top_k * 16 + (lane & 15)], wts[id] * acc[0][0][i], __ATOMIC_RELAXED,
                               __HIP_MEMORY_SCOPE_WORKGROUP);
      }
    }
    acc[0][0] = f32x4{0.f, 0.f, 0.f, 0.f};
  };
  if (i0 < i1) {
    S ring[D];
#pragma unroll
    for (int d = 0; d < D; ++d) {
      issue(ring[d], i0 + d);
      __builtin_amdgcn_sched_barrier(0);
    }
    int j = i0;
    for (; j + D < i1; j += D) {
#pragma unroll
      for (int d = 0; d < D; ++d) {
        consume(ring[d], j + d);
        issue(ring[d], j + D + d);
        __builtin_amdgcn_sched_barrier(0);
      }
    }
#pragma unroll
    for (int d = 0; d < D; ++d)
      if (j + d < i1) consume(ring[d], j + d);
  }
  __syncthreads();

  const int col = slab * 16;
  for (int i = threadIdx.x; i < a.N * 16; i += kDownWaves * kWave) {
    float y = 0.f;
#pragma unroll
    for (int w = 0; w < kDownWaves; ++w) y += lds[w * a.N * 16 + i];
    if (a.splits == 1) {
      static_cast<T*>(a.out)[static_cast<int64_t>(i >> 4) * a.os + col + (i & 15)] = from_f32<T>(y);
    } else {
      float* p = a.part + (static_cast<int64_t>(split) * a.N + (i >> 4)) * a.H + col + (i & 15);
      __hip_atomic_store(p, y, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
  }
  if (a.splits == 1) return;
  __builtin_amdgcn_s_waitcnt(0);
  __syncthreads();
  if (threadIdx.x == 0) {
    const uint32_t prev = __hip_atomic_fetch_add(a.counters + slab, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    last = prev == static_cast<uint32_t>(a.splits) - 1;
    if (last) __hip_atomic_store(a.counters + slab, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  __syncthreads();
  if (!last) return;
  for (int i = threadIdx.x; i < a.N * 16; i += kDownWaves * kWave) {
    const float* p = a.part + static_cast<int64_t>(i >> 4) * a.H + col + (i & 15);
    float y = 0.f;
    for (int s = 0; s < a.splits; ++s)
      y += __hip_atomic_load(p + static_cast<int64_t>(s) * a.N * a.H, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    static_cast<T*>(a.out)[static_cast<int64_t>(i >> 4) * a.os + col + (i & 15)] = from_f32<T>(y);
  }
}

// Groups of 16 that A assignments to E experts can form.
int64_t max_groups(int64_t A, int64_t E) { return std::min(A, std::min(A, E) + A / kMlTile); }

// Splits of the second kernel's work: enough workgroups to fill the chip.
int64_t down_splits(int64_t A, int64_t E, int64_t H, int64_t blocks) {
  const int64_t slabs = H / 16, cus = std::max(1, device_cu_count());
  const int64_t want = std::max<int64_t>(1, (2 * cus + slabs / 2) / slabs);
  const int64_t most = std::max<int64_t>(1, std::min(A, E) * blocks / (2 * kDownWaves));
  return std::min<int64_t>(kMlMaxSplits, std::min(want, most));
}

struct MlLayout {
  int64_t act, gexpert, glist, part, partial, counters;  // offsets, end of the partials, bytes of counters
};

MlLayout ml_layout(int64_t N, int64_t top_k, int64_t E, int64_t H, int64_t I, int64_t splits) {
  const int64_t A = N * top_k, g = max_groups(A, E);
  auto up = [](int64_t v) { return (v + 255) / 256 * 256; };
  MlLayout l;
  l.act = 0;
  l.gexpert = up(A * I * 2);
  l.glist = l.gexpert + up(4 * (g + 1));
  l.part = l.glist + up(4 * kMlTile * g);
  l.partial = l.part + (splits > 1 ? up(splits * N * H * 4) : 0);
  l.counters = up(H / 16 * 4);
  return l;
}

bool ml_sizes_ok(int64_t N, int64_t top_k, int64_t E, int64_t H, int64_t I) {
  return N >= 0 && N <= kMlMaxTokens && top_k >= 1 && N * top_k <= kMlMaxAssign && top_k <= kMlMaxAssign && E >= 1 &&
         E <= kMlMaxExperts && H >= 32 && I >= 32 && H % 32 == 0 && I % 32 == 0 && H <= (1 << 24) && I <= (1 << 24);
}

template <typename T, int GPB>
int ml_up(const MlArgs& a, hipStream_t s) {
  const dim3 grid(static_cast<unsigned>(max_groups(a.A, a.E) * a.slabs));
  k_moe_layer_up<T, GPB, 4><<<grid, kUpWaves * kWave, 0, s>>>(a);
  return launch_status();
}

template <typename T, int GPB>
int ml_down(const MlArgs& a, hipStream_t s) {
  const int64_t g = max_groups(a.A, a.E);
  const size_t lds = 4 * (size_t(kDownWaves) * a.N * 16 + a.A) + 2 * size_t(g) * (kMlTile + 1) + 16;
  k_moe_layer_down<T, GPB, 4><<<dim3(static_cast<unsigned>(a.slabs * a.splits)), kDownWaves * kWave, lds, s>>>(a);
  return launch_status();
}

template <typename T>
int ml_run(MlArgs a, int gpb1, int gpb2, hipStream_t s) {
  a.slabs = a.I / 16;
  int st;
  switch (gpb1) {
    case 0: st = ml_up<T, 0>(a, s); break;
    case 1: st = ml_up<T, 1>(a, s); break;
    case 2: st = ml_up<T, 2>(a, s); break;
    default: st = ml_up<T, 4>(a, s); break;
  }
  if (st != EMBER_OK) return st;
  a.slabs = a.H / 16;
  switch (gpb2) {
    case 0: return ml_down<T, 0>(a, s);
    case 1: return ml_down<T, 1>(a, s);
    case 2: return ml_down<T, 2>(a, s);
    default: return ml_down<T, 4>(a, s);
  }
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

int ml_call(const MlCall& c, const WeightView& w1, const WeightView& w2, int gpb1, int gpb2) {
  if (!ml_sizes_ok(c.N, c.top_k, c.E, c.H, c.I) || (c.dtype != EMBER_F16 && c.dtype != EMBER_BF16) ||
      (c.id_bytes != 4 && c.id_bytes != 8) || dtype_size(c.weight_dtype) == 0 || c.xs < 0 || c.os < 0)
    return EMBER_EINVAL;
  if (c.N == 0) return EMBER_OK;
  const int64_t splits = down_splits(c.N * c.top_k, c.E, c.H, w2.nb);
  const MlLayout l = ml_layout(c.N, c.top_k, c.E, c.H, c.I, splits);
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
  a.glist = reinterpret_cast<int*>(ws + l.glist);
  a.part = reinterpret_cast<float*>(ws + l.part);
  a.counters = reinterpret_cast<uint32_t*>(ws + c.workspace_bytes - l.counters);
  a.out = c.out;
  a.os = c.os;
  a.splits = static_cast<int>(splits);
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
  const MlLayout l = ml_layout(num_tokens, top_k, num_experts, hidden, inter, kMlMaxSplits);
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
    w1 = WeightView{w_gate_up, 2 * inter * hidden, kUnit, 1024, 512, inter / 64 * kUnit, 4096, 8, 128, 2,
                    static_cast<int>(hidden / 64)};
  }
  if (down_row_stride != 0) {
    w2 = rows_view(w_down, down_expert_stride, down_row_stride, 0, inter);
  } else {  // ember_moe_down_pack_weight's slabs
    const int64_t slab = 16 * inter;
    w2 = WeightView{w_down, hidden * inter, 4 * slab, slab, 0, 1024, 512, 8, 128, 1, static_cast<int>(inter / 64)};
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
  if (b1 < 0 || b2 < 0) return EMBER_EINVAL;
  WeightView w1{}, w2{};
  w1.w = packed_gate_up;
  w1.es = b1;
  w1.parts = 2;
  w1.nb = static_cast<int>(cdiv(hidden, kW4Block));
  w2.w = packed_down;
  w2.es = b2;
  w2.parts = 1;
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
