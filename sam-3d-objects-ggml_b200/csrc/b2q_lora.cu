// b2q_lora.cu -- low-rank adapters of many requests beside a shared projection:
//   y[t] = resid[t] + scale_g * B_g (A_g x[t]),  g = the adapter of row t
// (rows of no adapter: y[t] = resid[t]; a scale per row may come in beside the adapter's).
//
// Bound by the rows' bytes (x and resid read, y written) or, for single tokens, by
// latency.  h = A x enters the second product as a sum of 16-bit numbers (two, or
// three of bf16: the value, and what rounding it left) of a power of two per row, so
// neither fp16's range nor the 8 bits of bf16 limit it.  Products are m16n8k16; K and the rank are taken in an
// order that suits the loads: lane q of a quad has 8 consecutive values of every 32
// (4 of 16 where the rank is at most 16).
//
// Few rows per adapter: one launch, a cluster of 8 CTAs per tile of 16 sorted rows.
//   1  each CTA multiplies its eighth of K
//   2  the partial h meet in the CTAs' shared memories: each CTA adds up its own two
//      rows, scales them, and hands them to all eight
//   3  each CTA makes its eighth of the columns of y
// More rows: two launches over tiles of 64 sorted rows.  The first makes h (cp.async
// stages of x's and A's rows; where the tiles are few, a cluster shares out K and adds
// the parts up) in fp32 in the workspace; the second, launched early, streams y.
//
// Measured: 32 rows of 24 adapters, rank 16, 4096 -> 4096: 6.6 us, one chain of
// latencies; 8.7k rows of 7 adapters, rank 64, 4096 -> 6144, bf16: 106 us, 4530 GB/s
// (y's stages 32 columns wide instead of 64: 17 us more; read into registers instead: 30
// more; the parts of K added up by every CTA of the second launch instead: 3 to 5 more,
// 27 of 186 at rank 128; tiles of 128 rows in the first: 10 more).
#include "b2q_groups.cuh"
#include "b2q_internal.h"
#include "b2q_ptx.cuh"

#include <algorithm>

namespace b2q {

namespace {

constexpr int kRanks = 8;  // CTAs of a cluster
constexpr int kWarps = 8, kThreads = kWarps * 32;
constexpr int kStages = 4;
constexpr int kStageK = 64;

// RP: the rank, padded to 16, 32, 64 or 128.  Bytes of a row of h's 16-bit numbers: conflict-free reads.
template <int RP>
constexpr int kPitch = RP * 2 + (RP >= 64 ? 64 : 0);

// Numbers that make up one of h: 22 bits of fp16, 24 of bf16; 16 of bf16 where y has 8.  (8700 rows, 4096 x 6144, bf16, fp32
// y: rank 64 108 us and an error of 2.6e-7 with three, 99 us and 5.8e-7 with two; rank 128 196 and 4.7e-7, 169 and 9.3e-7.)
template <int X, int Y>
constexpr int kTerms = X == 2 && Y == 0 ? 3 : 2;

template <int X, int Y, int RP>
struct ClusterShape {
  static constexpr int M = 16;
  static constexpr int OFF_SUM = kWarps * 16 * RP * 4;  // behind the warps' parts: this CTA's h
  static constexpr int OFF_H = OFF_SUM + M * RP * 4;
  static constexpr int OFF_EXP = OFF_H + kTerms<X, Y> * M * kPitch<RP>;
  static constexpr int OFF_ROW = OFF_EXP + M * 4;
  static constexpr int SMEM = OFF_ROW + M * 4;
};
constexpr int kTile = 64;  // rows of the two-launch form
constexpr int kMaxSplits = 8;
template <int RP>
struct ShrinkShape {
  static constexpr int STAGE = (kTile + RP) * 128;
  static constexpr int PART = kWarps * 16 * RP * 4;
  static constexpr int OFF_ROW = kStages * STAGE > PART ? kStages * STAGE : PART;
  static constexpr int SMEM = OFF_ROW + kTile * 4;
};
template <int X, int Y, int RP>
struct ExpandShape {
  static constexpr int YS = Y == 0 ? 4 : 2;
  static constexpr int COLS = 64, STAGES = 3;  // of one stage of y's and B's columns
  static constexpr int YROW = COLS * YS, BROW = RP * 2;
  static constexpr int STAGE = kTile * YROW + COLS * BROW;
  static constexpr int OFF_H = STAGES * STAGE;
  static constexpr int OFF_EXP = OFF_H + kTerms<X, Y> * kTile * kPitch<RP>;
  static constexpr int OFF_ROW = OFF_EXP + kTile * 4;
  static constexpr int SMEM = OFF_ROW + kTile * 4;
};

template <int X>
__device__ __forceinline__ void mma16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (X == 2)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Two 16-bit numbers of type X in one word, and back.
template <int X>
__device__ __forceinline__ uint16_t bits16(float v) {
  if constexpr (X == 1) return __half_as_ushort(__float2half_rn(v));
  else return __bfloat16_as_ushort(__float2bfloat16_rn(v));
}
template <int X>
__device__ __forceinline__ float from16(uint16_t b) {
  if constexpr (X == 1) return __half2float(__ushort_as_half(b));
  else return __bfloat162float(__ushort_as_bfloat16(b));
}

// The rows of tile t: row_of[i], -1 where there is none.
template <int M>
__device__ __forceinline__ void tile_rows(const LoraArgs& p, const GroupTile& t, int* row_of) {
  for (int i = threadIdx.x; i < M; i += kThreads) {
    int r = -1;
    if (t.begin + i < t.end) {
      r = __ldg(p.order + t.begin + i);
      if (r < 0 || r >= p.T) r = -1;
    }
    row_of[i] = r;
  }
}

__device__ __forceinline__ float row_scale(const LoraArgs& p, int row) {
  return p.row_scales && row >= 0 ? __ldg(p.row_scales + row) : 1.0f;
}

// A row's PER rank values in a lane -> the 16-bit numbers that they are sums of, at most 1 in magnitude, pairs in a
// word; returns the power of two that they were divided by.  (fmaxf passes over NaN; a row with an infinity keeps its
// values.)  WIDTH neighbouring lanes have the row.
template <int X, int Y, int PER, int WIDTH>
__device__ __forceinline__ float split_row(const float (&v)[PER], uint32_t (&terms)[kTerms<X, Y>][PER / 2]) {
  float top = 0.0f;
#pragma unroll
  for (int e = 0; e < PER; ++e) top = fmaxf(top, fabsf(v[e]));
#pragma unroll
  for (int o = WIDTH / 2; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  int e2 = 0;
  if (top > 0.0f && top < INFINITY) frexpf(top, &e2);
  e2 = max(-126, min(126, e2));
  const float down = __int_as_float((127 - e2) << 23);
#pragma unroll
  for (int e = 0; e < PER; e += 2) {
    float w[2] = {v[e] * down, v[e + 1] * down};
    const bool finite[2] = {fabsf(w[0]) < INFINITY, fabsf(w[1]) < INFINITY};
#pragma unroll
    for (int s = 0; s < kTerms<X, Y>; ++s) {
      uint16_t h[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        h[i] = bits16<X>(w[i]);
        w[i] = finite[i] ? w[i] - from16<X>(h[i]) : 0.0f;  // exact
      }
      terms[s][e / 2] = h[0] | (static_cast<uint32_t>(h[1]) << 16);
    }
  }
  return __int_as_float((127 + e2) << 23);
}

// Columns [n0, n1) of y for 16 rows of a tile, 32 columns at a time from n0 + split * 32 on, every `step`-th of them.
// h: the lane's row of the 16-bit numbers (what rounding left lies `rest` bytes on, and so on); up: the powers of two of
// rows g and g + 8.  32 columns are two groups of 16: lane q has columns 4 q .. 4 q + 3 of a group (2 q and 2 q + 1
// of its two products), so y moves 4 values at a time.
template <int X, int Y, int RP>
__device__ __forceinline__ void stream_columns(const LoraArgs& p, int group, bool live, const uint8_t* h, int rest,
                                               float up_a, float up_b, int row_a, int row_b, int64_t n0, int64_t n1,
                                               int split, int step) {
  using YV = typename Val<Y>::type;
  const int lane = threadIdx.x & 31, g = lane >> 2, q = lane & 3;
  const uint16_t* b = static_cast<const uint16_t*>(p.b) + static_cast<int64_t>(live ? group : 0) * p.N * p.rank;
  const float up[2] = {up_a, up_b};
  constexpr int YS = static_cast<int>(sizeof(YV));
  const bool aligned = (reinterpret_cast<uintptr_t>(p.resid) | reinterpret_cast<uintptr_t>(p.y) |
                        static_cast<uintptr_t>(p.ldr * YS) | static_cast<uintptr_t>(p.ldy * YS)) % (4 * YS) == 0;
  const bool have[2] = {row_a >= 0, row_b >= 0};
  const YV* from[2] = {static_cast<const YV*>(p.resid) + (have[0] ? row_a : 0) * p.ldr + 4 * q,
                       static_cast<const YV*>(p.resid) + (have[1] ? row_b : 0) * p.ldr + 4 * q};
  YV* to[2] = {static_cast<YV*>(p.y) + (have[0] ? row_a : 0) * p.ldy + 4 * q,
               static_cast<YV*>(p.y) + (have[1] ? row_b : 0) * p.ldy + 4 * q};
  float y[2][2][4];  // [row][group of 16 columns]
  auto read = [&](int64_t n) {
    const bool full = aligned && n + 32 <= n1;
#pragma unroll
    for (int r = 0; r < 2; ++r)
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        if (full && have[r]) {
          load_vec<Y>(from[r] + n + u * 16, y[r][u]);
        } else {
#pragma unroll
          for (int i = 0; i < 4; ++i)
            y[r][u][i] = have[r] && n + u * 16 + 4 * q + i < n1 ? Val<Y>::load(from[r] + n + u * 16 + i) : 0.0f;
        }
      }
  };
  if (n0 + split * 32 < n1) read(n0 + split * 32);
  const int col_of = 4 * (g >> 1) + (g & 1);  // column of a group that lane row g brings; 2 more in the second product
  for (int64_t n = n0 + split * 32; n < n1; n += step) {
    float acc[4][4] = {};
    if (live) {
      const uint16_t* bn = b + (n + col_of) * p.rank;
      const int left = static_cast<int>(min(n1 - n, int64_t{32})) - col_of;
#pragma unroll
      for (int kb = 0; kb < (RP == 16 ? 1 : RP / 32); ++kb) {
        const int k = RP == 16 ? q * 4 : kb * 32 + q * 8;
        uint4 w[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int c = (j >> 1) * 16 + (j & 1) * 2;
          w[j] = make_uint4(0, 0, 0, 0);
          if (c < left && k < p.rank) {
            if constexpr (RP == 16) {
              const uint2 v = __ldg(reinterpret_cast<const uint2*>(bn + c * p.rank + k));
              w[j].x = v.x, w[j].y = v.y;
            } else {
              w[j] = __ldg(reinterpret_cast<const uint4*>(bn + c * p.rank + k));
            }
          }
        }
#pragma unroll
        for (int s = 0; s < kTerms<X, Y>; ++s) {  // the numbers, then what rounding them left
          const uint8_t* hs = h + s * rest + k * 2;
          if constexpr (RP == 16) {
            const uint2 u = *reinterpret_cast<const uint2*>(hs), v = *reinterpret_cast<const uint2*>(hs + 8 * kPitch<RP>);
            const uint32_t a0[4] = {u.x, v.x, u.y, v.y};
#pragma unroll
            for (int j = 0; j < 4; ++j) mma16<X>(acc[j], a0, w[j].x, w[j].y);
          } else {
            const uint4 u = *reinterpret_cast<const uint4*>(hs), v = *reinterpret_cast<const uint4*>(hs + 8 * kPitch<RP>);
            const uint32_t a0[4] = {u.x, v.x, u.y, v.y}, a1[4] = {u.z, v.z, u.w, v.w};
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              mma16<X>(acc[j], a0, w[j].x, w[j].y);
              mma16<X>(acc[j], a1, w[j].z, w[j].w);
            }
          }
        }
      }
    }
    float out[2][2][4];
#pragma unroll
    for (int r = 0; r < 2; ++r)
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int i = 0; i < 4; ++i)  // (rows of no adapter stay as they are, to the bit)
          out[r][u][i] = live ? fmaf(up[r], acc[2 * u + (i >> 1)][2 * r + (i & 1)], y[r][u][i]) : y[r][u][i];
    // The next columns' values are asked for before these are written (y may be resid: other columns).
    if (n + step < n1) read(n + step);
    const bool full = aligned && n + 32 <= n1;
#pragma unroll
    for (int r = 0; r < 2; ++r)
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        if (!have[r]) continue;
        if (full) {
          store_vec<Y>(to[r] + n + u * 16, out[r][u]);
        } else {
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (n + u * 16 + 4 * q + i < n1) to[r][n + u * 16 + i] = Val<Y>::to(out[r][u][i]);
        }
      }
  }
}

template <int X, int Y, int RP>
__global__ void __launch_bounds__(kThreads, RP <= 64 ? 2 : 1) lora_cluster_kernel(const LoraArgs p) {
  using Sh = ClusterShape<X, Y, RP>;
  constexpr int M = Sh::M, N8 = RP / 8;
  extern __shared__ __align__(1024) uint8_t smem[];
  float* part = reinterpret_cast<float*>(smem);
  float* sum = reinterpret_cast<float*>(smem + Sh::OFF_SUM);
  float* power = reinterpret_cast<float*>(smem + Sh::OFF_EXP);
  int* row_of = reinterpret_cast<int*>(smem + Sh::OFF_ROW);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int g = lane >> 2, q = lane & 3;
  const int rank = static_cast<int>(cluster_ctarank());

  grid_wait();
  const GroupTile t = find_group_tile(p.offsets, p.groups, p.T, blockIdx.x / kRanks, M);
  if (t.group < 0) return;  // (all eight CTAs)
  const bool live = t.group < p.groups;
  if (!live && p.resid == p.y) return;
  tile_rows<M>(p, t, row_of);
  __syncthreads();
  const int row_a = row_of[g], row_b = row_of[g + 8];

  if (live) {
    // ------------------------------------------------------ 1: this CTA's eighth of K
    const int64_t k_slice = ((p.K + kRanks - 1) / kRanks + 31) / 32 * 32;
    const int64_t k0 = min(p.K, rank * k_slice), k1 = min(p.K, k0 + k_slice);
    const uint16_t* x = static_cast<const uint16_t*>(p.x);
    const uint16_t* a = static_cast<const uint16_t*>(p.a) + static_cast<int64_t>(t.group) * p.rank * p.K;
    float acc[N8][4] = {};
    const uint16_t* xa = x + (row_a < 0 ? 0 : row_a) * p.ldx + q * 8;
    const uint16_t* xb = x + (row_b < 0 ? 0 : row_b) * p.ldx + q * 8;
#pragma unroll 2
    for (int64_t k = k0 + warp * 32; k < k1; k += kWarps * 32) {
      const bool in = k + q * 8 < k1;
      const uint4 zero = make_uint4(0, 0, 0, 0);
      const uint4 u = in && row_a >= 0 ? __ldg(reinterpret_cast<const uint4*>(xa + k)) : zero;
      const uint4 v = in && row_b >= 0 ? __ldg(reinterpret_cast<const uint4*>(xb + k)) : zero;
      uint4 w[N8];
#pragma unroll
      for (int j = 0; j < N8; ++j)
        w[j] = in && j * 8 < p.rank ? __ldg(reinterpret_cast<const uint4*>(a + (j * 8 + g) * p.K + k + q * 8)) : zero;
      const uint32_t a0[4] = {u.x, v.x, u.y, v.y}, a1[4] = {u.z, v.z, u.w, v.w};
#pragma unroll
      for (int j = 0; j < N8; ++j) {
        mma16<X>(acc[j], a0, w[j].x, w[j].y);
        mma16<X>(acc[j], a1, w[j].z, w[j].w);
      }
    }
#pragma unroll
    for (int j = 0; j < N8; ++j) {
      float* d = part + (warp * 16 + g) * RP + j * 8 + 2 * q;
      *reinterpret_cast<float2*>(d) = make_float2(acc[j][0], acc[j][1]);
      *reinterpret_cast<float2*>(d + 8 * RP) = make_float2(acc[j][2], acc[j][3]);
    }
    __syncthreads();
    for (int i = threadIdx.x; i < M * RP / 4; i += kThreads) {
      float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
      for (int s = 0; s < kWarps; ++s) {
        const float4 w = *reinterpret_cast<const float4*>(part + s * 16 * RP + i * 4);
        v.x += w.x, v.y += w.y, v.z += w.z, v.w += w.w;
      }
      *reinterpret_cast<float4*>(sum + i * 4) = v;
    }
    // (asked for before the others are waited for)
    constexpr int MINE = M / kRanks;
    float scale = p.scales ? __ldg(p.scales + t.group) : 1.0f;
    if (p.row_scales && warp < MINE) scale *= row_scale(p, row_of[rank * MINE + warp]);
    cluster_sync();
    // --------------------------- 2: this CTA's rows, from all eight and to all eight
    constexpr int PER = RP >= 64 ? RP / 32 : 2, LANES = RP / PER;  // rows; values of a lane
    static_assert(MINE <= kWarps, "a row a warp");
    if (warp < MINE) {
      const int m = rank * MINE + warp;
      float v[PER] = {};
      if (lane * PER < p.rank) {  // (what an infinite x makes of A's missing rows is no number)
#pragma unroll
        for (int s = 0; s < kRanks; ++s) {
          const uint32_t from = cluster_addr(sum + m * RP + lane * PER, s);
#pragma unroll
          for (int e = 0; e < PER; e += 2) {
            float2 w;
            asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(w.x), "=f"(w.y) : "r"(from + e * 4) : "memory");
            v[e] += w.x;
            v[e + 1] += w.y;
          }
        }
      }
#pragma unroll
      for (int e = 0; e < PER; ++e) v[e] *= scale;
      uint32_t terms[kTerms<X, Y>][PER / 2];
      const float up = split_row<X, Y, PER, 32>(v, terms);
#pragma unroll
      for (int s = 0; s < kRanks; ++s) {
        if (lane < LANES) {
          const uint32_t to = cluster_addr(smem + Sh::OFF_H + m * kPitch<RP> + lane * PER * 2, s);
#pragma unroll
          for (int k = 0; k < kTerms<X, Y>; ++k)
#pragma unroll
            for (int e = 0; e < PER / 2; ++e)
              asm volatile("st.shared::cluster.b32 [%0], %1;" ::"r"(to + k * M * kPitch<RP> + e * 4), "r"(terms[k][e]) : "memory");
        }
        if (lane == 0)
          asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(cluster_addr(power + m, s)), "f"(up) : "memory");
      }
    }
    cluster_sync();
  }
  // -------------------------------------------- 3: this CTA's eighth of the columns
  const int64_t n_slice = ((p.N + kRanks - 1) / kRanks + 31) / 32 * 32;
  const int64_t n0 = min(p.N, rank * n_slice), n1 = min(p.N, n0 + n_slice);
  stream_columns<X, Y, RP>(p, t.group, live, smem + Sh::OFF_H + g * kPitch<RP>, M * kPitch<RP>, live ? power[g] : 0.0f,
                           live ? power[g + 8] : 0.0f, row_a, row_b, n0, n1, warp, kWarps * 32);
}

// h of one tile of 64 sorted rows, K shared out over a cluster of p.splits CTAs: p.part [T][RP], rows in sorted order.
template <int X, int RP>
__global__ void __launch_bounds__(kThreads) lora_shrink_kernel(const LoraArgs p) {
  using Sh = ShrinkShape<RP>;
  constexpr int N8 = RP / 8, ROWS = kTile + RP, PIECES = (ROWS * 8 + kThreads - 1) / kThreads;
  extern __shared__ __align__(1024) uint8_t smem[];
  int* row_of = reinterpret_cast<int*>(smem + Sh::OFF_ROW);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int g = lane >> 2, q = lane & 3;
  const int rg = warp & 3, half = warp >> 2;  // 16 rows, and 32 of a stage's 64 of K
  const int split = blockIdx.x % p.splits;
  grid_wait();
  const GroupTile t = find_group_tile(p.offsets, p.groups, p.T, blockIdx.x / p.splits, kTile);
  if (t.group >= 0 && t.group < p.groups) {
    tile_rows<kTile>(p, t, row_of);
    __syncthreads();
    const int64_t k_slice = ((p.K + p.splits - 1) / p.splits + kStageK - 1) / kStageK * kStageK;
    const int64_t k0 = min(p.K, split * k_slice), k1 = min(p.K, k0 + k_slice);
    const uint16_t* x = static_cast<const uint16_t*>(p.x);
    const uint16_t* a = static_cast<const uint16_t*>(p.a) + static_cast<int64_t>(t.group) * p.rank * p.K;
    // x's rows and A's rows, 64 of K a stage; odd rows have their halves swapped.
    const uint32_t base = smem_u32(smem);
    const uint16_t* src[PIECES];
    bool there[PIECES];
    const int c = threadIdx.x & 7;
#pragma unroll
    for (int i = 0; i < PIECES; ++i) {
      const int r = (threadIdx.x >> 3) + i * (kThreads / 8);
      src[i] = x;
      there[i] = false;
      if (r < kTile) {
        there[i] = row_of[r] >= 0;
        if (there[i]) src[i] = x + row_of[r] * p.ldx;
      } else if (r < ROWS && r - kTile < p.rank) {
        there[i] = true;
        src[i] = a + static_cast<int64_t>(r - kTile) * p.K;
      }
    }
    int stage_in = 0;
    int64_t k_in = k0;
    auto ask = [&]() {
      if (k_in < k1) {
#pragma unroll
        for (int i = 0; i < PIECES; ++i) {
          const int r = (threadIdx.x >> 3) + i * (kThreads / 8);
          if (r < ROWS) {
            const bool in = there[i] && k_in + c * 8 < k1;
            cp16(base + stage_in * Sh::STAGE + r * 128 + ((c ^ ((r & 1) << 2)) << 4), src[i] + (in ? k_in + c * 8 : 0), in);
          }
        }
        k_in += kStageK;
      }
      asm volatile("cp.async.commit_group;" ::: "memory");
      stage_in = stage_in + 1 == kStages ? 0 : stage_in + 1;
    };
    for (int i = 0; i < kStages - 1; ++i) ask();
    float acc[N8][4] = {};
    int stage = 0;
    for (int64_t k = k0; k < k1; k += kStageK) {
      asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 2) : "memory");
      __syncthreads();  // the stage has arrived, and the one before it has been read
      ask();
      const uint8_t* sp = smem + stage * Sh::STAGE + (((half * 4 + q) ^ ((g & 1) << 2)) << 4);
      const uint4 u = *reinterpret_cast<const uint4*>(sp + (rg * 16 + g) * 128);
      const uint4 v = *reinterpret_cast<const uint4*>(sp + (rg * 16 + g + 8) * 128);
      const uint32_t a0[4] = {u.x, v.x, u.y, v.y}, a1[4] = {u.z, v.z, u.w, v.w};
#pragma unroll
      for (int j = 0; j < N8; ++j) {
        const uint4 w = *reinterpret_cast<const uint4*>(sp + (kTile + j * 8 + g) * 128);
        mma16<X>(acc[j], a0, w.x, w.y);
        mma16<X>(acc[j], a1, w.z, w.w);
      }
      stage = stage + 1 == kStages ? 0 : stage + 1;
    }
    __syncthreads();  // the stages become the halves' sums
    float* part = reinterpret_cast<float*>(smem);
#pragma unroll
    for (int j = 0; j < N8; ++j) {
      float* d = part + (warp * 16 + g) * RP + j * 8 + 2 * q;
      *reinterpret_cast<float2*>(d) = make_float2(acc[j][0], acc[j][1]);
      *reinterpret_cast<float2*>(d + 8 * RP) = make_float2(acc[j][2], acc[j][3]);
    }
    // A cluster's CTAs have the parts of K of one tile: each adds up a share of it, parts in order.
    if (p.splits > 1) cluster_sync();
    else __syncthreads();
    float* out = p.part + t.begin * static_cast<int64_t>(RP);
    for (int i = split * kThreads + threadIdx.x; i < (t.end - t.begin) * RP / 4; i += p.splits * kThreads) {
      float4 w[kMaxSplits][2];
#pragma unroll
      for (int s = 0; s < kMaxSplits; ++s)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          w[s][h] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
          if (s < p.splits)
            asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                         : "=f"(w[s][h].x), "=f"(w[s][h].y), "=f"(w[s][h].z), "=f"(w[s][h].w)
                         : "r"(cluster_addr(part + h * kTile * RP + i * 4, s))
                         : "memory");
        }
      float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
      for (int s = 0; s < kMaxSplits; ++s)
#pragma unroll
        for (int h = 0; h < 2; ++h) v.x += w[s][h].x, v.y += w[s][h].y, v.z += w[s][h].z, v.w += w[s][h].w;
      if (p.row_scales) {  // (here and not in the second launch, whose loads it would hold up: 2.3 of 108 us)
        const float own = row_scale(p, row_of[i * 4 / RP]);
        v.x *= own, v.y *= own, v.z *= own, v.w *= own;
      }
      *reinterpret_cast<float4*>(out + i * 4) = v;
    }
    if (p.splits > 1) cluster_sync();  // (nobody leaves before all have read)
  }
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}

// One of p.slices parts of the columns of y for a tile of 64 sorted rows.  Whole
// groups of 64 columns come in cp.async stages (resid's values and B's rows, each
// brought once for all warps); a warp has 16 rows and 32 of the columns.  What is
// left, or lies on addresses that cp.async does not take, is read straight.
template <int X, int Y, int RP>
__global__ void __launch_bounds__(kThreads, 2) lora_expand_kernel(const LoraArgs p) {
  using YV = typename Val<Y>::type;
  constexpr int YS = static_cast<int>(sizeof(YV));
  using Sh = ExpandShape<X, Y, RP>;
  extern __shared__ __align__(1024) uint8_t smem[];
  uint8_t* hs = smem + Sh::OFF_H;
  float* power = reinterpret_cast<float*>(smem + Sh::OFF_EXP);
  int* row_of = reinterpret_cast<int*>(smem + Sh::OFF_ROW);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int g = lane >> 2, q = lane & 3;
  const int rg = warp & 3, half = warp >> 2;
  const GroupTile t = find_group_tile(p.offsets, p.groups, p.T, blockIdx.x / p.slices, kTile);
  const bool live = t.group >= 0 && t.group < p.groups;
  // The first launch had waited for all before it when it let this one begin, so only its results are waited for:
  // by the tiles that need them, and by all others too, so that this launch does not end before it.
  if (!live) grid_wait();
  if (t.group < 0 || (!live && p.resid == p.y)) return;
  tile_rows<kTile>(p, t, row_of);
  __syncthreads();
  const int count = t.end - t.begin;
  const int64_t n_slice = ((p.N + p.slices - 1) / p.slices + Sh::COLS - 1) / Sh::COLS * Sh::COLS;
  const int64_t n0 = min(p.N, (blockIdx.x % p.slices) * n_slice), n1 = min(p.N, n0 + n_slice);
  const bool aligned = (reinterpret_cast<uintptr_t>(p.resid) | reinterpret_cast<uintptr_t>(p.y) |
                        static_cast<uintptr_t>(p.ldr * YS) | static_cast<uintptr_t>(p.ldy * YS)) % 16 == 0;
  const int whole = live && aligned ? static_cast<int>((n1 - n0) / Sh::COLS) : 0;
  const uint16_t* b = static_cast<const uint16_t*>(p.b) + (static_cast<int64_t>(live ? t.group : 0) * p.N + n0) * p.rank;

  // What a thread fetches of a stage: 16-byte pieces of y's rows and of B's.
  constexpr int YP = Sh::YROW / 16, BP = Sh::BROW / 16;          // pieces of a row
  constexpr int YN = kTile * YP / kThreads, BN = (Sh::COLS * BP + kThreads - 1) / kThreads;
  static_assert(kTile * YP % kThreads == 0, "");
  const uint32_t base = smem_u32(smem);
  const YV* ysrc[YN];
  bool yhave[YN];
#pragma unroll
  for (int i = 0; i < YN; ++i) {
    const int at = threadIdx.x + i * kThreads, r = row_of[at / YP];
    yhave[i] = r >= 0;
    ysrc[i] = static_cast<const YV*>(p.resid) + (r < 0 ? 0 : r) * p.ldr + n0 + at % YP * (16 / YS);
  }
  const uint16_t* bsrc[BN];
  bool bhave[BN];
#pragma unroll
  for (int i = 0; i < BN; ++i) {
    const int at = threadIdx.x + i * kThreads, r = at / BP, c = at % BP;
    bhave[i] = c * 8 < p.rank && r < Sh::COLS;
    bsrc[i] = b + (bhave[i] ? r * p.rank + c * 8 : 0);
  }
  int next = 0, put = 0;
  auto ask = [&]() {
    if (next < whole) {
      const uint32_t to = base + put * Sh::STAGE;
#pragma unroll
      for (int i = 0; i < YN; ++i) {
        const int at = threadIdx.x + i * kThreads, r = at / YP, c = at % YP;
        cp16(to + r * Sh::YROW + ((c ^ ((r & 1) << 2)) << 4), ysrc[i], yhave[i]);
        ysrc[i] += Sh::COLS;
      }
#pragma unroll
      for (int i = 0; i < BN; ++i) {
        const int at = threadIdx.x + i * kThreads, r = at / BP, c = at % BP;
        if (Sh::COLS * BP % kThreads == 0 || r < Sh::COLS)
          cp16(to + kTile * Sh::YROW + r * Sh::BROW + ((BP >= 8 ? c ^ ((r & 1) << 2) : c) << 4), bsrc[i], bhave[i]);
        bsrc[i] += Sh::COLS * p.rank;
      }
      ++next;
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
    put = put + 1 == Sh::STAGES ? 0 : put + 1;
  };
  for (int i = 0; i < Sh::STAGES - 1; ++i) ask();  // (these do not depend on the first launch)

  if (live) {
    const float scale = p.scales ? __ldg(p.scales + t.group) : 1.0f;
    grid_wait();
    constexpr int LANES = RP / 4;  // of a row, 4 values each
#pragma unroll
    for (int i = 0; i < kTile * LANES / kThreads; ++i) {
      const int at = i * kThreads + threadIdx.x, m = at / LANES, c = at % LANES;
      float v[4] = {};
      if (m < count && c * 4 < p.rank) {  // (what an infinite x makes of A's missing rows is no number)
        const float4* from = reinterpret_cast<const float4*>(p.part + (t.begin + m) * static_cast<int64_t>(RP)) + c;
        const float4 w = *from;
        v[0] = w.x, v[1] = w.y, v[2] = w.z, v[3] = w.w;
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] *= scale;
      uint32_t terms[kTerms<X, Y>][2];
      const float up = split_row<X, Y, 4, LANES>(v, terms);
      uint2* to = reinterpret_cast<uint2*>(hs + m * kPitch<RP>) + c;
#pragma unroll
      for (int k = 0; k < kTerms<X, Y>; ++k) to[k * (kTile * kPitch<RP> / 8)] = make_uint2(terms[k][0], terms[k][1]);
      if (c == 0) power[m] = up;
    }
  }
  __syncthreads();
  const int m = rg * 16 + g;
  const int row_a = row_of[m], row_b = row_of[m + 8];
  const float up_a = live ? power[m] : 0.0f, up_b = live ? power[m + 8] : 0.0f;
  const uint8_t* h = hs + m * kPitch<RP>;
  constexpr int REST = kTile * kPitch<RP>;
  constexpr int HALF = Sh::COLS / 2, UNITS = HALF / 16;  // a warp's columns, and groups of 16 of them
  YV* ta = static_cast<YV*>(p.y) + (row_a < 0 ? 0 : row_a) * p.ldy + n0 + half * HALF + 4 * q;
  YV* tb = static_cast<YV*>(p.y) + (row_b < 0 ? 0 : row_b) * p.ldy + n0 + half * HALF + 4 * q;
  const int col = half * HALF + 4 * (g >> 1) + (g & 1);  // of B, and 2 more in the second product
  const int flip = (g & 1) << 2;
  int take = 0;
  for (int i = 0; i < whole; ++i) {
    asm volatile("cp.async.wait_group %0;" ::"n"(Sh::STAGES - 2) : "memory");
    __syncthreads();  // the stage has arrived, and the one before it has been read
    ask();
    const uint8_t* sp = smem + take * Sh::STAGE;
    const uint8_t* bp = sp + kTile * Sh::YROW + col * Sh::BROW;
    float acc[2 * UNITS][4] = {};
#pragma unroll
    for (int kb = 0; kb < (RP == 16 ? 1 : RP / 32); ++kb) {
      uint4 w[2 * UNITS];
#pragma unroll
      for (int j = 0; j < 2 * UNITS; ++j) {
        const uint8_t* at = bp + ((j >> 1) * 16 + (j & 1) * 2) * Sh::BROW;  // (columns of the same parity)
        if constexpr (RP == 16) {
          const uint2 v = *reinterpret_cast<const uint2*>(at + q * 8);
          w[j] = make_uint4(v.x, v.y, 0, 0);
        } else {
          w[j] = *reinterpret_cast<const uint4*>(at + ((BP >= 8 ? (kb * 4 + q) ^ flip : kb * 4 + q) << 4));
        }
      }
#pragma unroll
      for (int s = 0; s < kTerms<X, Y>; ++s) {  // the numbers, then what rounding them left
        if constexpr (RP == 16) {
          const uint2 u = *reinterpret_cast<const uint2*>(h + s * REST + q * 8);
          const uint2 v = *reinterpret_cast<const uint2*>(h + s * REST + 8 * kPitch<RP> + q * 8);
          const uint32_t a0[4] = {u.x, v.x, u.y, v.y};
#pragma unroll
          for (int j = 0; j < 2 * UNITS; ++j) mma16<X>(acc[j], a0, w[j].x, w[j].y);
        } else {
          const uint4 u = *reinterpret_cast<const uint4*>(h + s * REST + kb * 64 + q * 16);
          const uint4 v = *reinterpret_cast<const uint4*>(h + s * REST + 8 * kPitch<RP> + kb * 64 + q * 16);
          const uint32_t a0[4] = {u.x, v.x, u.y, v.y}, a1[4] = {u.z, v.z, u.w, v.w};
#pragma unroll
          for (int j = 0; j < 2 * UNITS; ++j) {
            mma16<X>(acc[j], a0, w[j].x, w[j].y);
            mma16<X>(acc[j], a1, w[j].z, w[j].w);
          }
        }
      }
    }
#pragma unroll
    for (int u = 0; u < UNITS; ++u) {
      float ya[4], yb[4];
      const int c = half * HALF + u * 16 + 4 * q, piece = c * YS / 16;
      const int yc = ((piece ^ flip) << 4) + c * YS % 16;
      load_vec<Y>(reinterpret_cast<const YV*>(sp + m * Sh::YROW + yc), ya);
      load_vec<Y>(reinterpret_cast<const YV*>(sp + (m + 8) * Sh::YROW + yc), yb);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        ya[e] = fmaf(up_a, acc[2 * u + (e >> 1)][e & 1], ya[e]);
        yb[e] = fmaf(up_b, acc[2 * u + (e >> 1)][2 + (e & 1)], yb[e]);
      }
      if (row_a >= 0) store_vec<Y>(ta + u * 16, ya);
      if (row_b >= 0) store_vec<Y>(tb + u * 16, yb);
    }
    ta += Sh::COLS;
    tb += Sh::COLS;
    take = take + 1 == Sh::STAGES ? 0 : take + 1;
  }
  asm volatile("cp.async.wait_all;" ::: "memory");
  if (rg * 16 >= count) return;
  stream_columns<X, Y, RP>(p, t.group, live, h, REST, up_a, up_b, row_a, row_b, n0 + static_cast<int64_t>(whole) * Sh::COLS,
                           n1, half, 2 * 32);
}

int padded(int rank) { return rank <= 16 ? 16 : rank <= 32 ? 32 : rank <= 64 ? 64 : 128; }
int64_t tiles_of(const LoraArgs& a, int rows) { return a.T / rows + std::min<int64_t>(a.groups + 1, a.T); }
// One launch while its tiles of 16 rows are few; many adapters cost it half a tile each and the two launches most of
// a tile of 64.  Measured, one launch against two, 2048 x 2048 and 4096 x 6144 (us): rank 64, 512 rows of 16 adapters
// 14/16 and 30/28, 768 of 16 17/16 and 32/30, 768 of 64 26/30 and 48/59, 1536 of 64 37/31 and 65/57; rank 16, 768 rows of
// 16 10/11 and 20/19, 1024 of 16 15/13 and 29/25, 1024 of 64 17/17 and 32/37; rank 128, 256 rows of 16 20/20 and 40/44,
// 512 of 16 30/22 and 59/46, 512 of 64 58/53 and 101/104.
bool two_launches(int64_t T, int groups, int rank) {
  return T / 16 > (rank > 64 ? 20 : (rank > 16 ? 36 : 44) + std::min<int64_t>(groups, T) / 2);
}

// Parts of K of the first launch, the CTAs of a cluster: up to three CTAs an SM, or two of the 96 KB ones of rank 128,
// where tiles are few.  Measured (8700 rows, bf16), rank 64, 4096 -> 4096 of 32 adapters: with three or four 95 us, with
// two 102; 4096 x 6144 of 7: with two or three 108, with four 112; 2000 rows of 8, 2048 x 2048, fp16: with two 19.6, with three
// 21.0.  Rank 128, 2000 rows of 8, 2048 x 2048: with two 37.4, with three 39.3.
int splits_of(int64_t T, int64_t K, int groups, int rank, int num_sms) {
  const int64_t tiles = T / kTile + std::min<int64_t>(groups, T);
  const int64_t most = std::min<int64_t>({kMaxSplits, (rank <= 64 ? 3 : 2) * num_sms / tiles, K / 256});
  return most >= 8 ? 8 : most >= 4 ? 4 : most >= 2 ? 2 : 1;
}

template <int X, int Y, int RP>
cudaError_t launch_shape(LoraArgs a, int num_sms, cudaStream_t s) {
  if (!two_launches(a.T, a.groups, a.rank)) {
    using Sh = ClusterShape<X, Y, RP>;
    constexpr auto k = lora_cluster_kernel<X, Y, RP>;
    if (cudaError_t e = allow_smem<k>(Sh::SMEM)) return e;
    const int64_t tiles = tiles_of(a, Sh::M);
    if (tiles > INT32_MAX / kRanks) return cudaErrorInvalidValue;
    return launch_early(k, dim3(static_cast<unsigned>(tiles * kRanks)), dim3(kThreads), Sh::SMEM, s, kRanks, a);
  }
  constexpr auto shrink = lora_shrink_kernel<X, RP>;
  constexpr auto expand = lora_expand_kernel<X, Y, RP>;
  constexpr int expand_smem = ExpandShape<X, Y, RP>::SMEM;
  if (cudaError_t e = allow_smem<shrink>(ShrinkShape<RP>::SMEM)) return e;
  if (cudaError_t e = allow_smem<expand>(expand_smem)) return e;
  const int64_t tiles = tiles_of(a, kTile);
  a.splits = splits_of(a.T, a.K, a.groups, a.rank, num_sms);
  // (and the parts of the columns of the second, of at least 256: 128 cost 31 -> 34 us at 4096 rows of 16 adapters, rank
  // 64, 2048 x 2048.  5 CTAs an SM against 6: 105 us against 109 for the 8.7k rows above, 77 against 73 for rank 16.)
  a.slices = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>((5 * num_sms + tiles - 1) / tiles, (a.N + 255) / 256)));
  if (tiles > INT32_MAX / std::max(a.splits, a.slices)) return cudaErrorInvalidValue;
  if (cudaError_t e = launch_early(shrink, dim3(static_cast<unsigned>(tiles * a.splits)), dim3(kThreads), ShrinkShape<RP>::SMEM,
                                   s, a.splits, a))
    return e;
  return launch_early(expand, dim3(static_cast<unsigned>(tiles * a.slices)), dim3(kThreads), expand_smem, s, 1, a);
}

template <int X, int Y>
cudaError_t launch_types(const LoraArgs& a, int num_sms, cudaStream_t s) {
  switch (padded(a.rank)) {
    case 16: return launch_shape<X, Y, 16>(a, num_sms, s);
    case 32: return launch_shape<X, Y, 32>(a, num_sms, s);
    case 64: return launch_shape<X, Y, 64>(a, num_sms, s);
    default: return launch_shape<X, Y, 128>(a, num_sms, s);
  }
}

}  // namespace

size_t lora_workspace(int64_t T, int groups, int rank) {
  if (T <= 0 || !two_launches(T, groups, rank)) return 0;
  return static_cast<size_t>(T) * padded(rank) * 4;
}

cudaError_t launch_lora(const LoraArgs& a, int xtype, int ytype, int num_sms, cudaStream_t s) {
  if (xtype == kXF16) return ytype == kXF32 ? launch_types<1, 0>(a, num_sms, s) : launch_types<1, 1>(a, num_sms, s);
  return ytype == kXF32 ? launch_types<2, 0>(a, num_sms, s) : launch_types<2, 2>(a, num_sms, s);
}

}  // namespace b2q
