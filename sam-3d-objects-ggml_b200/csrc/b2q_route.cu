// b2q_route.cu -- the router of an expert layer and the plan of rows that go by
// group.
//
//   key_e = logit_e + bias_e, or score_e + bias_e with the softmax or sigmoid scores; the `top` largest keys, ties to
//   the lower expert
//   w_j   = softmax or sigmoid of the chosen logits, times scale
//   order   = the slots (token * top + choice) sorted by expert, stable
//   offsets = where each expert's slots begin
//
// A row's experts are spread over the lanes of one warp and stay in registers,
// as unsigned numbers that order as the keys do (-0 as 0, NaN as -infinity); up to 8
// of a lane are sorted first.  Each choice is one warp maximum (redux) of the lanes'
// largest and, among the lanes that hold it, one minimum of the expert's number;
// its lane then moves on to its next largest.
//
// The sort is a counting sort without float work or global atomics: every CTA
// counts the experts of its run of slots; then every CTA adds up the counts of
// all runs itself (the L2 serves them), so none waits for another, and places
// its slots: the warps take consecutive parts of the run, ranks inside a warp
// come from the lanes that hold the same expert.  The second launch is made
// early (programmatic dependent launch).  Where one CTA can do it all, it does:
// one launch.
//
// Measured: 12 tokens, 6 of 64 experts: 4.6 us, one CTA's chain; 20471 tokens, 8 of 160:
// 23.5 us, 600 instructions a row in two thirds of the issue slots (a thread a row
// with its choices in registers: 49 us for the first launch instead of 22); with the
// bias on the scores 26.1 (sigmoid) and 29.3 (softmax).  More than 256 experts are not
// sorted first, and those of more than 512 (32 a lane) do not all stay in registers:
// 20000 tokens, 8 of 256, 512, 1024: 32, 59, 276 us.
#include "b2q_groups.cuh"
#include "b2q_internal.h"

#include <algorithm>

namespace b2q {

namespace {

constexpr int kWarps = 32, kThreads = kWarps * 32;
constexpr int kMaxRuns = 148;
// Rows of logits that a CTA has, at least (a row a warp), and up to which one CTA does everything: twice as many where a
// row is little work.  Measured, one launch against two (us): 64 rows of 64 experts, one, two and eight choices 6.0/6.7,
// 6.4/6.9, 8.1/7.7; 48 of 256, eight 12.1/10.5; 64 of 1024, one 47/27.  At least 32 rows a CTA against 64 and 128: 512 rows
// of 64 experts, eight choices 8.2, 10.2, 15.1; 4736 of 256 14.1, 18.9, 29.4; 2048 of 1024 61, 108, 195.
constexpr int kRouteRun = 32;
int route_one(int E, int top) { return E <= 64 && top <= 4 ? 64 : 32; }
// Slots of given groups, the same.  One launch against two: 2000 slots of 8, 64, 256 and 1024 groups 4.3/5.3, 5.9/5.8,
// 6.4/6.7, 9.2/12.3; 3000 4.9/5.4, 7.2/5.9, 7.9/6.9, 10.7/12.5.  At least 512 slots a CTA against 256 and 1024: 8192 of 64
// groups 6.1, 6.5, 6.8; of 1024 13.6, 16.6, 13.7.
constexpr int kRowsRun = 512, kRowsOne = 2048;

__device__ __forceinline__ uint32_t key_bits(float v) {
  if (v != v) v = -INFINITY;
  const uint32_t b = __float_as_uint(v + 0.0f);  // -0 becomes 0
  return b ^ ((b >> 31) ? 0xffffffffu : 0x80000000u);
}
constexpr uint32_t kKeyNone = 0x007fffffu;  // of -infinity; all others are larger

// Counts the groups of slots [s0, s1) warp by warp into counts[warp][groups + 1].
__device__ __forceinline__ void warp_part(int s0, int s1, int* lo, int* hi) {
  const int each = ((s1 - s0 + kWarps - 1) / kWarps + 31) / 32 * 32;
  *lo = min(s1, s0 + static_cast<int>(threadIdx.x >> 5) * each);
  *hi = min(s1, *lo + each);
}

__device__ __forceinline__ int group_of(const int32_t* ids, int s, int groups) {
  const int g = ids[s];
  return (g < 0 || g >= groups) ? groups : g;
}

// Exclusive scan over the block of the sums that thread t holds of its `n`
// consecutive values; `sums` has kWarps + 1 ints.
__device__ __forceinline__ int block_exclusive(int v, int* sums) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int inc = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int u = __shfl_up_sync(0xffffffffu, inc, o);
    if (lane >= o) inc += u;
  }
  if (lane == 31) sums[warp] = inc;
  __syncthreads();
  int before = 0;
  for (int w = 0; w < warp; ++w) before += sums[w];
  __syncthreads();
  return before + inc - v;
}

// Places the slots of run `run` of `runs`; run_counts [runs][groups + 1] of all
// runs, or nullptr when this run is all there is.  smem: (kWarps + 1) * (groups
// + 1) + kWarps ints.
__device__ void place_run(const int32_t* ids, int S, int groups, int run, int runs, int run_slots,
                          const int32_t* run_counts, int32_t* order, int32_t* offsets, int* smem) {
  const int G = groups + 1;
  int* counts = smem;               // [kWarps][G]
  int* base = smem + kWarps * G;    // [G]
  int* sums = base + G;             // [kWarps]
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int s0 = static_cast<int>(min(static_cast<int64_t>(run) * run_slots, static_cast<int64_t>(S)));
  const int s1 = static_cast<int>(min(static_cast<int64_t>(s0) + run_slots, static_cast<int64_t>(S)));
  int lo, hi;
  warp_part(s0, s1, &lo, &hi);
  for (int i = threadIdx.x; i < kWarps * G; i += kThreads) counts[i] = 0;
  __syncthreads();
  for (int s = lo + lane; s < hi; s += 32) atomicAdd(&counts[warp * G + group_of(ids, s, groups)], 1);
  __syncthreads();
  // Totals of every group, and of the runs before this one: a warp a run, its lanes the groups.
  int* total = sums + kWarps;
  for (int g = threadIdx.x; g < G; g += kThreads) {
    int c = 0;
    if (!run_counts)
      for (int w = 0; w < kWarps; ++w) c += counts[w * G + g];
    total[g] = c;
    base[g] = 0;
  }
  __syncthreads();
  if (run_counts) {
    // (six groups of a lane and five runs asked for at a time)
    for (int g0 = lane; g0 < G; g0 += 6 * 32) {
      int all[6] = {}, before[6] = {};
      for (int r0 = warp; r0 < runs; r0 += 5 * kWarps) {
        int c[5][6];
#pragma unroll
        for (int i = 0; i < 5; ++i)
#pragma unroll
          for (int j = 0; j < 6; ++j) {
            const int r = r0 + i * kWarps, g = g0 + 32 * j;
            c[i][j] = r < runs && g < G ? __ldg(run_counts + static_cast<int64_t>(r) * G + g) : 0;
          }
#pragma unroll
        for (int i = 0; i < 5; ++i)
#pragma unroll
          for (int j = 0; j < 6; ++j) {
            all[j] += c[i][j];
            if (r0 + i * kWarps < run) before[j] += c[i][j];
          }
      }
#pragma unroll
      for (int j = 0; j < 6; ++j)
        if (g0 + 32 * j < G) {
          atomicAdd(&total[g0 + 32 * j], all[j]);
          atomicAdd(&base[g0 + 32 * j], before[j]);
        }
    }
    __syncthreads();
  }
  const int each = (G + kThreads - 1) / kThreads;
  int mine = 0;
  for (int i = 0; i < each; ++i) {
    const int g = threadIdx.x * each + i;
    if (g < G) mine += total[g];
  }
  int at = block_exclusive(mine, sums);
  for (int i = 0; i < each; ++i) {
    const int g = threadIdx.x * each + i;
    if (g >= G) break;
    if (run == 0) offsets[g] = at;
    int place = at + base[g];
    at += total[g];
    for (int w = 0; w < kWarps; ++w) {  // where each warp's slots of this group begin
      const int c = counts[w * G + g];
      counts[w * G + g] = place;
      place += c;
    }
  }
  __syncthreads();
  for (int s = lo; s < hi; s += 32) {
    const bool there = s + lane < hi;
    const int g = there ? group_of(ids, s + lane, groups) : -1;
    const unsigned same = __match_any_sync(0xffffffffu, g);
    const int rank = __popc(same & ((1u << lane) - 1));
    int place = 0;
    if (there) place = counts[warp * G + g] + rank;
    __syncwarp();
    if (there && rank == 0) counts[warp * G + g] += __popc(same);
    __syncwarp();
    if (there) order[place] = s + lane;
  }
}

constexpr size_t place_smem(int groups) { return (static_cast<size_t>(kWarps + 2) * (groups + 1) + kWarps) * 4; }

// NV: experts of a lane.  ON_SCORE: the bias is added to the scores.  (A kernel of its own: the scores of all experts
// before the choice are work that the others do not have.)
template <int T, int NV, bool ON_SCORE>
__global__ void __launch_bounds__(kThreads) route_kernel(const RouteArgs a) {
  extern __shared__ int smem[];
  using V = typename Val<T>::type;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int E = a.E;
  const bool one = a.run_counts == nullptr;
  grid_wait();
  if (!one) {
    for (int i = threadIdx.x; i <= E; i += kThreads) smem[i] = 0;
    __syncthreads();
  }
  const int64_t t0 = static_cast<int64_t>(blockIdx.x) * a.run_rows;
  const int64_t t1 = min(t0 + a.run_rows, a.T);
  float x[NV], next[NV];
  auto fetch = [&](int64_t t) {
    const V* row = static_cast<const V*>(a.logits) + t * a.ld;
#pragma unroll
    for (int i = 0; i < NV; ++i) next[i] = lane + 32 * i < E ? Val<T>::load(row + lane + 32 * i) : -INFINITY;
  };
  if (t0 + warp < t1) fetch(t0 + warp);
  for (int64_t t = t0 + warp; t < t1; t += kWarps) {
    uint32_t key[NV];
    if constexpr (ON_SCORE) {
      float m = -INFINITY, z = 0.0f;  // of the softmax, as for the weights below
      if (a.scoring == 0) {
#pragma unroll
        for (int i = 0; i < NV; ++i) m = fmaxf(m, next[i]);  // (fmaxf passes over NaN)
#pragma unroll
        for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
#pragma unroll
        for (int i = 0; i < NV; ++i)
          if (next[i] > -INFINITY) z += next[i] == m ? 1.0f : expf(next[i] - m);
#pragma unroll
        for (int o = 16; o; o >>= 1) z += __shfl_xor_sync(0xffffffffu, z, o);
      }
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        x[i] = next[i];
        const int e = lane + 32 * i;
        key[i] = 0u;
        if (x[i] > -INFINITY) {  // (neither NaN nor an expert behind the last)
          const float score = a.scoring == 1 ? 1.0f / (1.0f + expf(-x[i])) : (x[i] == m ? 1.0f : expf(x[i] - m)) / z;
          key[i] = key_bits(score + __ldg(a.bias + e));
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        x[i] = next[i];
        const int e = lane + 32 * i;
        key[i] = e < E ? key_bits(a.bias ? x[i] + __ldg(a.bias + e) : x[i]) : 0u;
      }
    }
    if (t + kWarps < t1) fetch(t + kWarps);
    float picked = 0.0f;  // lane j: the logit of choice j
    int chosen = -1;
    if constexpr (NV <= 8) {
      // The lane's keys in falling order, equal ones in the experts' order (neighbours change places only where the
      // later is larger), with their places as digits of `places`: a choice takes the first and moves the others up.
      uint32_t places = 0x76543210u;
#pragma unroll
      for (int n = 0; n < NV; ++n)
#pragma unroll
        for (int i = n & 1; i + 1 < NV; i += 2) {
          const bool change = key[i + 1] > key[i];
          const uint32_t high = max(key[i], key[i + 1]), low = min(key[i], key[i + 1]);
          key[i] = high;
          key[i + 1] = low;
          const uint32_t differ = ((places >> 4) ^ places) & (0xfu << (4 * i));  // of the two digits
          places ^= change ? differ | (differ << 4) : 0u;
        }
      for (int j = 0; j < a.top; ++j) {
        const uint32_t top = __reduce_max_sync(0xffffffffu, key[0]);
        if (top <= kKeyNone) break;  // only -infinity is left
        const unsigned mine = lane + 32 * (places & 15u);
        const unsigned e = __reduce_min_sync(0xffffffffu, key[0] == top ? mine : 0x7fffffffu);
        const bool taken = mine == e;
#pragma unroll
        for (int i = 0; i + 1 < NV; ++i) key[i] = taken ? key[i + 1] : key[i];
        key[NV - 1] = taken ? 0u : key[NV - 1];
        places = taken ? places >> 4 : places;
        chosen = lane == j ? static_cast<int>(e) : chosen;
      }
    } else {
      for (int j = 0; j < a.top; ++j) {
        uint32_t best = key[0];
#pragma unroll
        for (int i = 1; i < NV; ++i) best = max(best, key[i]);
        const uint32_t top = __reduce_max_sync(0xffffffffu, best);
        if (top <= kKeyNone) break;
        unsigned mine = 0x7fffffffu;  // the lane's lowest expert with that key
#pragma unroll
        for (int i = NV - 1; i >= 0; --i)
          if (key[i] == top) mine = lane + 32 * i;
        const int e = static_cast<int>(__reduce_min_sync(0xffffffffu, mine));
#pragma unroll
        for (int i = 0; i < NV; ++i) key[i] = e == lane + 32 * i ? 0u : key[i];
        chosen = lane == j ? e : chosen;
      }
    }
    const bool there = chosen >= 0;
    // lane j: the logit of choice j, from the lane that has it
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const float v = __shfl_sync(0xffffffffu, x[i], chosen & 31);
      if (chosen >> 5 == i) picked = v;
    }
    float w = 0.0f;
    if (a.scoring == 1) {
      if (there) w = 1.0f / (1.0f + expf(-picked));
    } else {
      // the largest logit of all (of the choice, when only the choice counts); its own weight is e^0, also where it is infinite
      float m = there ? picked : -INFINITY;
      if (!a.renorm) {
#pragma unroll
        for (int i = 0; i < NV; ++i) m = fmaxf(m, x[i]);  // (fmaxf passes over NaN)
      }
#pragma unroll
      for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
      if (there) w = picked == m ? 1.0f : expf(picked - m);
      if (!a.renorm) {
        float z = 0.0f;
#pragma unroll
        for (int i = 0; i < NV; ++i)
          if (lane + 32 * i < E && x[i] == x[i]) z += x[i] == m ? 1.0f : expf(x[i] - m);
#pragma unroll
        for (int o = 16; o; o >>= 1) z += __shfl_xor_sync(0xffffffffu, z, o);
        if (there) w /= z;
      }
    }
    if (a.renorm) {
      float z = w;
#pragma unroll
      for (int o = 16; o; o >>= 1) z += __shfl_xor_sync(0xffffffffu, z, o);
      w = z > 0.0f ? w / z : 0.0f;
    }
    if (lane < a.top) {
      a.ids[t * a.top + lane] = chosen;
      a.weights[t * a.top + lane] = w * a.scale;
      if (!one) atomicAdd(&smem[there ? chosen : E], 1);
    }
  }
  __syncthreads();
  if (one) {
    place_run(a.ids, static_cast<int>(a.T * a.top), E, 0, 1, static_cast<int>(a.T * a.top), nullptr, a.order,
              a.offsets, smem);
  } else {
    for (int i = threadIdx.x; i <= E; i += kThreads)
      a.run_counts[static_cast<int64_t>(blockIdx.x) * (E + 1) + i] = smem[i];
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  }
}

__global__ void __launch_bounds__(kThreads) count_kernel(const int32_t* ids, int S, int groups, int run_slots,
                                                         int32_t* run_counts) {
  extern __shared__ int smem[];
  grid_wait();
  for (int i = threadIdx.x; i <= groups; i += kThreads) smem[i] = 0;
  __syncthreads();
  const int64_t s0 = static_cast<int64_t>(blockIdx.x) * run_slots;
  const int64_t s1 = min(s0 + run_slots, static_cast<int64_t>(S));
  for (int64_t s = s0 + threadIdx.x; s < s1; s += kThreads) atomicAdd(&smem[group_of(ids, static_cast<int>(s), groups)], 1);
  __syncthreads();
  for (int i = threadIdx.x; i <= groups; i += kThreads)
    run_counts[static_cast<int64_t>(blockIdx.x) * (groups + 1) + i] = smem[i];
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}

__global__ void __launch_bounds__(kThreads) place_kernel(const int32_t* ids, int S, int groups, int run_slots,
                                                         const int32_t* run_counts, int32_t* order, int32_t* offsets) {
  extern __shared__ int smem[];
  grid_wait();
  place_run(ids, S, groups, blockIdx.x, gridDim.x, run_slots, run_counts, order, offsets, smem);
}

cudaError_t launch_place(const int32_t* ids, int64_t S, int groups, int runs, int run_slots, const int32_t* run_counts,
                         int32_t* order, int32_t* offsets, cudaStream_t s) {
  const size_t smem = place_smem(groups);
  // (always the most that any call needs: calls of other sizes from other threads share the setting)
  if (cudaError_t e = allow_smem<place_kernel>(place_smem(kMaxGroups))) return e;
  return launch_early(place_kernel, dim3(static_cast<unsigned>(runs)), dim3(kThreads), smem, s, 1, ids, static_cast<int>(S),
                      groups, run_slots, run_counts, order, offsets);
}

// y [T * top] rows -> out [T] rows: out = resid + sum_j w_j y_j, choices in
// order.  A thread has N columns of one token and asks for four choices' values
// at a time.  Bound by the bytes of y.
template <int Y, int O, int N>
__global__ void __launch_bounds__(256) combine_kernel(const CombineArgs a) {
  using YV = typename Val<Y>::type;
  using OV = typename Val<O>::type;
  const int64_t t = static_cast<int64_t>(blockIdx.x) * blockDim.y + threadIdx.y;
  const int64_t n = (static_cast<int64_t>(blockIdx.y) * blockDim.x + threadIdx.x) * N;
  grid_wait();
  if (t >= a.T || n >= a.n) return;
  float sum[N] = {};
  Raw<O, N> more;
  if (a.resid) more = load_raw<O, N>(static_cast<const OV*>(a.resid) + t * a.ldr + n);
  const YV* y = static_cast<const YV*>(a.y) + t * a.top * a.ldy + n;
  const float* w = a.weights + t * a.top;
  const int32_t* ids = a.ids ? a.ids + t * a.top : nullptr;
  for (int j0 = 0; j0 < a.top; j0 += 4) {
    Raw<Y, N> raw[4];
    float share[4];
    bool there[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      there[j] = j0 + j < a.top && !(ids && __ldg(ids + j0 + j) < 0);
      if (there[j]) {
        share[j] = __ldg(w + j0 + j);
        raw[j] = load_raw<Y, N>(y + (j0 + j) * a.ldy);
      }
    }
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (there[j]) {
        float v[N];
        from_raw<Y, N>(raw[j], v);
#pragma unroll
        for (int i = 0; i < N; ++i) sum[i] = fmaf(share[j], v[i], sum[i]);
      }
  }
  if (a.resid) {
    float v[N];
    from_raw<O, N>(more, v);
#pragma unroll
    for (int i = 0; i < N; ++i) sum[i] += v[i];
  }
  store_vec<O>(static_cast<OV*>(a.out) + t * a.ldo + n, sum);
}

}  // namespace

namespace {
RunPlan plan_of(int64_t units, int one, int least) {
  RunPlan p;
  if (units <= one) return p;
  const int64_t runs = std::min<int64_t>(kMaxRuns, (units + least - 1) / least);
  p.run_units = static_cast<int>((units + runs - 1) / runs);
  p.runs = static_cast<int>((units + p.run_units - 1) / p.run_units);
  return p;
}
}  // namespace

RunPlan route_plan(int64_t T, int64_t E, int64_t top) {
  return plan_of(T, route_one(static_cast<int>(E), static_cast<int>(top)), kRouteRun);
}
RunPlan rows_plan(int64_t S) { return plan_of(S, kRowsOne, kRowsRun); }

cudaError_t launch_route(RouteArgs a, int type, cudaStream_t s) {
  const RunPlan p = route_plan(a.T, a.E, a.top);
  const bool one = p.runs == 1;
  a.run_rows = one ? a.T : p.run_units;
  const size_t smem = one ? place_smem(a.E) : (a.E + 1) * 4;
  if (one) a.run_counts = nullptr;
  auto run = [&](auto ty) {
    constexpr int T = decltype(ty)::value;
    const int nv = (a.E + 31) / 32;
    auto go = [&](auto nv_c, auto on) {
      constexpr auto k = route_kernel<T, decltype(nv_c)::value, decltype(on)::value>;
      if (cudaError_t e = allow_smem<k>(place_smem(kMaxGroups))) return e;
      return launch_early(k, dim3(static_cast<unsigned>(p.runs)), dim3(kThreads), smem, s, 1, a);
    };
    auto shape = [&](auto on) {
      if (nv <= 1) return go(std::integral_constant<int, 1>(), on);
      if (nv <= 2) return go(std::integral_constant<int, 2>(), on);
      if (nv <= 3) return go(std::integral_constant<int, 3>(), on);
      if (nv <= 4) return go(std::integral_constant<int, 4>(), on);
      if (nv <= 5) return go(std::integral_constant<int, 5>(), on);
      if (nv <= 6) return go(std::integral_constant<int, 6>(), on);
      if (nv <= 8) return go(std::integral_constant<int, 8>(), on);
      if (nv <= 16) return go(std::integral_constant<int, 16>(), on);
      return go(std::integral_constant<int, 32>(), on);
    };
    return a.on_score ? shape(std::true_type()) : shape(std::false_type());
  };
  const cudaError_t err = type == kXF32 ? run(std::integral_constant<int, 0>())
                          : type == kXF16 ? run(std::integral_constant<int, 1>()) : run(std::integral_constant<int, 2>());
  if (err != cudaSuccess || one) return err;
  return launch_place(a.ids, a.T * a.top, a.E, p.runs, p.run_units * a.top, a.run_counts, a.order, a.offsets, s);
}

cudaError_t launch_group_rows(const int32_t* ids, int64_t S, int groups, int32_t* order, int32_t* offsets,
                              int32_t* run_counts, cudaStream_t s) {
  const RunPlan p = rows_plan(S);
  if (p.runs == 1)
    return launch_place(ids, S, groups, 1, static_cast<int>(std::max<int64_t>(S, 1)), nullptr, order, offsets, s);
  if (cudaError_t e = launch_early(count_kernel, dim3(static_cast<unsigned>(p.runs)), dim3(kThreads), (groups + 1) * 4, s, 1, ids,
                                   static_cast<int>(S), groups, p.run_units, run_counts))
    return e;
  return launch_place(ids, S, groups, p.runs, p.run_units, run_counts, order, offsets, s);
}

cudaError_t launch_combine(const CombineArgs& a, int ytype, int otype, cudaStream_t s) {
  // N columns a thread where every row starts on them, else one.  8 of 16 bits; 4 where a type has 32.
  const int wide = ytype == kXF32 || otype == kXF32 ? 4 : 8;
  const int ys = ytype == kXF32 ? 4 : 2, os = otype == kXF32 ? 4 : 2;
  auto on = [&](const void* p, int64_t ld, int size) {
    return (reinterpret_cast<uintptr_t>(p) | static_cast<uintptr_t>(ld * size)) % (wide * size) == 0;
  };
  const bool vec = a.n % wide == 0 && on(a.y, a.ldy, ys) && on(a.out, a.ldo, os) && (!a.resid || on(a.resid, a.ldr, os));
  const int n = vec ? wide : 1;
  const int64_t cols = (a.n + n - 1) / n;
  int tx = 32;
  while (tx < 128 && tx < cols) tx *= 2;
  const dim3 block(tx, 256 / tx);
  const dim3 grid(static_cast<unsigned>((a.T + block.y - 1) / block.y), static_cast<unsigned>((cols + tx - 1) / tx));
  auto pick = [&](auto y, auto o) {
    constexpr int Y = decltype(y)::value, O = decltype(o)::value, N = Y == 0 || O == 0 ? 4 : 8;
    return launch_early(vec ? combine_kernel<Y, O, N> : combine_kernel<Y, O, 1>, grid, block, 0, s, 1, a);
  };
  auto pick_o = [&](auto y) {
    return otype == kXF32   ? pick(y, std::integral_constant<int, 0>())
           : otype == kXF16 ? pick(y, std::integral_constant<int, 1>())
                            : pick(y, std::integral_constant<int, 2>());
  };
  return ytype == kXF32   ? pick_o(std::integral_constant<int, 0>())
         : ytype == kXF16 ? pick_o(std::integral_constant<int, 1>())
                          : pick_o(std::integral_constant<int, 2>());
}

}  // namespace b2q
