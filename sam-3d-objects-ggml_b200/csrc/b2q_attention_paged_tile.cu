// b2q_attention_paged_tile.cu -- the paged attention (b2q_attention_paged.cu has
// its definition) for chunks of new tokens: more rows than the keys' bytes can
// pay for, so bound by the tensor cores and the exponentials.
//
// One CTA per SM takes 2 x 128 rows of one (request, kv head): two query tiles
// of floor(128 / G) tokens x G heads each, and walks the keys in tiles of 64:
//   warp 0       producer: Q once; K and V tiles into two rings, one TMA box per
//                page and 64 columns, issued by as many lanes.  Pages that are
//                absent, or past the length, are boxes outside the tensor: zeros
//   warps 1, 2   the MMAs of query tile 0 and 1, one thread each: S_i = Q_i K^T (M 128,
//                N 64, K D) and O_i += P_i V (M 128, N D, K 64; P from tensor memory).
//                One thread polling for both was the limit: 1177 us where two take 993
//   warp 3       V of the edge tiles (below)
//   warpgroups 1, 2: softmax of query tile 0 and 1, one row per thread: mask,
//                maximum, exp2, P rounded to the cache's type into tensor memory,
//                row sum of the unrounded P; the maximum in use is raised, and O
//                rescaled, only when a tile exceeds it by 2^8
// P rounded to 16 bits once, as the dense F16 attention has it: on random values
// that costs as much accuracy as rounding the output does, and a second P V for
// what it leaves would cost half the tensor time.
// Tensor memory: O_i (D columns each), and two 64-column buffers of S per query
// tile; P takes the place of its S.  So the next S of a query tile is computed
// while its softmax works on this one, and a softmax warp never waits for a round
// trip through the tensor pipe.  With tiles of 128 keys there is room for one S a
// query tile only: S, softmax and P V then follow one another (1027 us).
// Measured on two chunks of 3.9k tokens over 4k and 7.5k cached, 32 / 8 heads of
// 128: 985 us, 1020 TFLOP/s (1130 us at the clock that the power cap leaves in steady
// calls), the tensor pipe active half of the time; the
// softmax warps' own chain (loads from tensor memory, maximum, exps, stores) is
// what a tile waits for.
//
// Edge tiles -- not every row sees every key -- are masked in the scores.  Their V
// may hold an infinity or a NaN in keys that some rows do not see, and P = 0
// does not cover those.  Warp 3 zeroes V rows that no row of the CTA sees,
// looks the rest of an edge tile's rows through, and takes non-finite ones out of
// the product; the rows that do see such a key add its share themselves, at the
// end, from global memory.
#include "b2q_paged.cuh"
#include "b2q_ptx.cuh"

#include <cmath>

namespace b2q {

namespace {

__device__ unsigned int g_paged_status = 0;

constexpr int kPtThreads = 384;
constexpr int kPtLaunchRegs = 168, kPtRegsControl = 56, kPtRegsSoftmax = 224;
static_assert(128 * kPtRegsControl + 256 * kPtRegsSoftmax <= kPtThreads * kPtLaunchRegs, "register split");
constexpr int kQHalf = 128 * 128, kHalf = kTileKeys * 128;  // bytes of 64 columns of Q, and of K or V
constexpr int kPolyPairs = 1;     // of every 4 pairs of exps, on the FMA pipe (the chunks above: 0 1076 us, 1 993, 2 1005)
constexpr int kMaxEdges = 24;     // edge tiles of a CTA that can hold non-finite keys

template <int D>
struct PtShape {
  static constexpr int HALVES = D / 64;
  static constexpr int QTILE = HALVES * kQHalf, TILE = HALVES * kHalf;
  static constexpr int STAGES = D == 64 ? 8 : 4;           // of the K ring and of the V ring
  // TMEM columns: S (and P) of query tile i, buffer x at S + 128 i + 64 x; O_i at O + D i
  static constexpr uint32_t S = 0, O = 256;
  static constexpr int Q_OFF = 0;
  static constexpr int K_OFF = 2 * QTILE, V_OFF = K_OFF + STAGES * TILE;
  static constexpr int BAR_OFF = V_OFF + STAGES * TILE;
  static constexpr int NBAR = 1 + 5 * STAGES + 12 + 4;
  static constexpr int MISC_OFF = BAR_OFF + NBAR * 8;
  // tmem holder, abort flag, number of bad tiles; bad tile numbers, bad key masks
  static constexpr int BYTES = MISC_OFF + 16 + kMaxEdges * (4 + 16) + 1024;
};

// Row r of a query tile is token r / G, head r % G.
struct PtMaps {
  CUtensorMap q, k, v;
};

template <bool BF16>
constexpr uint32_t idesc_16(int m, int n) {
  return idesc_f16(m, n) | (BF16 ? (1u << 7) | (1u << 10) : 0u);
}

// Shared-memory descriptor of V as an MN-major operand (128-byte swizzle): 64-column
// atoms `lbo` bytes apart, groups of 8 keys 1024 bytes apart.
__device__ __forceinline__ uint64_t pt_desc_v(uint32_t addr, uint32_t lbo) {
  uint64_t d = 0;
  d |= static_cast<uint64_t>((addr >> 4) & 0x3fffu);
  d |= static_cast<uint64_t>((lbo >> 4) & 0x3fffu) << 16;
  d |= static_cast<uint64_t>(1024u >> 4) << 32;
  d |= static_cast<uint64_t>(1u) << 46;
  d |= static_cast<uint64_t>(2u) << 61;
  return d;
}

// exp2 of a pair on the FMA pipe (the dense F16 attention has the derivation:
// Cody-Waite, cubic of least maximum relative error 7.5e-5); the others go to
// the MUFU.  Below -125, so for masked scores too, it is exactly 0: the cubic gives
// its constant term times 2^-125 there, which is subtracted.  bf16 holds 2^-125, and a
// row that sees no key would have become a mean of values that it must not see.
__device__ __forceinline__ float2 pt_ex2_poly(float2 x) {
  constexpr float kRound = 12582912.0f;
  const float2 one = make_float2(1.0f, 1.0f), neg = make_float2(-1.0f, -1.0f);
  x = make_float2(fmaxf(x.x, -125.0f), fmaxf(x.y, -125.0f));
  const float2 r = ffma2(x, one, make_float2(kRound, kRound));
  const float2 n = ffma2(r, one, make_float2(-kRound, -kRound));
  const float2 f = ffma2(n, neg, x);
  float2 q = ffma2(make_float2(0.0551716685f, 0.0551716685f), f, make_float2(0.242611140f, 0.242611140f));
  q = ffma2(q, f, make_float2(0.693260968f, 0.693260968f));
  constexpr float c0 = 0.999928057f, least = -c0 * 0x1p-125f;
  q = ffma2(q, f, make_float2(c0, c0));
  q = make_float2(__uint_as_float(__float_as_uint(q.x) + (__float_as_uint(r.x) << 23)),
                  __uint_as_float(__float_as_uint(q.y) + (__float_as_uint(r.y) << 23)));
  return ffma2(q, one, make_float2(least, least));
}

__device__ __forceinline__ float pt_max3(float a, float b, float c) {
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));  // a NaN score stays one
  return r;
}

// The key tiles of one query tile, and their places in the CTA's list.
struct TileList {
  int su, wu, hu;
  __device__ __forceinline__ int at(int j) const { return j < su ? j : wu + (j - su); }
  __device__ __forceinline__ int before(int kt) const {  // its tiles below kt
    return min(kt, su) + max(0, min(kt, hu) - wu);
  }
  __device__ __forceinline__ int count() const { return su + (hu - wu); }
};
__device__ __forceinline__ TileList list_of(const Units& u) {
  return {static_cast<int>(u.su), static_cast<int>(u.wu), static_cast<int>(u.hu)};
}

template <int D, bool BF16>
__global__ void __launch_bounds__(kPtThreads, 1)
    paged_tile_kernel(const __grid_constant__ PtMaps maps, const PagedArgs a, const int tok /* tokens of a query tile */) {
  using S = PtShape<D>;
  constexpr int ST = S::STAGES, HV = S::HALVES;
  extern __shared__ uint8_t pt_smem_raw[];
  const int b = blockIdx.z, hk = blockIdx.y;
  const int ntile = gridDim.x / a.splits;
  // the last tokens see the most keys: first
  const int tile = ntile - 1 - static_cast<int>(blockIdx.x) / a.splits, split = static_cast<int>(blockIdx.x) % a.splits;
  const Request rq = request_of(a, b);
  const int64_t i0 = static_cast<int64_t>(tile) * 2 * tok;
  if (i0 >= rq.n) return;
  const int nq = i0 + tok < rq.n ? 2 : 1;
  const int64_t i_end = min(rq.n, i0 + 2 * tok);
  const int64_t p_lo = rq.first + i0, p_hi = rq.first + i_end - 1;

  // Key tiles: the CTA's (both query tiles') and each query tile's; this split's stretch [u0, u1).
  const TileList all = list_of(units_of(a, rq.len, p_lo, p_hi, kTileKeys));
  const int u_all = all.count();
  const int u0 = static_cast<int>(min(static_cast<int64_t>(split) * a.split_units, static_cast<int64_t>(u_all)));
  const int u1 = split == a.splits - 1 ? u_all
                                       : static_cast<int>(min(static_cast<int64_t>(u_all), u0 + a.split_units));
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");  // the joining kernel may get ready
  if (split > 0 && u0 >= u_all) {  // no keys in this stretch
    for (int64_t r = threadIdx.x; r < (i_end - i0) * a.G; r += kPtThreads)
      a.part_ml[((rq.t0 + i0 + r / a.G) * a.Hq + static_cast<int64_t>(hk) * a.G + r % a.G) * a.splits + split] =
          make_float2(-INFINITY, 0.0f);
    return;
  }
  TileList own[2];  // of the whole range of keys
  int j0[2], j1[2];  // and those of the stretch
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    if (i < nq) {
      const int64_t f = i0 + i * tok, l = min(rq.n, f + tok) - 1;
      own[i] = list_of(units_of(a, rq.len, rq.first + f, rq.first + l, kTileKeys));
      j0[i] = u0 < u_all ? own[i].before(all.at(u0)) : own[i].count();
      j1[i] = u1 < u_all ? own[i].before(all.at(u1)) : own[i].count();
    } else {
      own[i] = {0, 0, 0};
      j0[i] = j1[i] = 0;
    }
  }
  const int nu = u1 - u0;
  const int64_t key_end = a.causal ? min(rq.len, p_hi + 1) : rq.len;
  // every row of the CTA sees every key of tile kt (absent pages aside)
  auto plain = [&](int kt) {
    const int64_t k0 = static_cast<int64_t>(kt) * kTileKeys, k1 = k0 + kTileKeys - 1;
    return k1 < rq.len && (!a.causal || k1 <= p_lo) && (a.window <= 0 || k0 > p_hi - a.window || k1 < a.sinks);
  };

  uint8_t* smem = pt_smem_raw + ((1024u - (smem_u32(pt_smem_raw) & 1023u)) & 1023u);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + S::BAR_OFF);
  uint64_t* q_full = bars;
  uint64_t* k_full = bars + 1;
  uint64_t* k_empty = k_full + ST;
  uint64_t* v_full = k_empty + ST;
  uint64_t* v_ok = v_full + ST;      // V landed and looked through
  uint64_t* v_empty = v_ok + ST;
  uint64_t* s_full = v_empty + ST;   // [query tile][buffer]
  uint64_t* p_full = s_full + 4;     // [query tile][buffer]
  uint64_t* pv_full = p_full + 4;    // [query tile][buffer]
  uint64_t* o_full = pv_full + 4;    // [query tile] all of P V, once
  uint64_t* done = o_full + 2;
  uint32_t* misc = reinterpret_cast<uint32_t*>(smem + S::MISC_OFF);
  uint32_t* tmem_holder = misc;
  volatile int* abort_flag = reinterpret_cast<volatile int*>(misc + 1);
  uint32_t* n_edges = misc + 2;
  uint32_t* bad_kt = misc + 4;       // [kMaxEdges]
  uint32_t* bad = bad_kt + kMaxEdges;  // [kMaxEdges][4] keys taken out of the product
  unsigned int* status = &g_paged_status;
  const int32_t* table = a.table + static_cast<int64_t>(b) * a.ldt;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int box = min(1 << a.page_shift, kTileKeys);  // keys of one TMA box
  const int boxes = kTileKeys / box;

  if (threadIdx.x == 0) {
    mbar_init(q_full, 1);
    for (int s = 0; s < ST; ++s) {
      mbar_init(&k_full[s], 1);
      mbar_init(&k_empty[s], nq);   // one per query tile
      mbar_init(&v_full[s], 1);
      mbar_init(&v_ok[s], 1);
      mbar_init(&v_empty[s], nq);
    }
    for (int x = 0; x < 4; ++x) {
      mbar_init(&s_full[x], 1);
      mbar_init(&p_full[x], 4);   // one arrival per softmax warp
      mbar_init(&pv_full[x], 1);
    }
    mbar_init(&o_full[0], 1);
    mbar_init(&o_full[1], 1);
    mbar_init(&done[0], 1);
    mbar_init(&done[1], 1);
    *abort_flag = 0;
    *n_edges = 0;
    fence_mbarrier_init();
  }
  for (int x = threadIdx.x; x < kMaxEdges * 5; x += kPtThreads) bad_kt[x] = 0;
  if (warp == 0 && lane < 3) tma_prefetch_desc(lane == 0 ? &maps.q : lane == 1 ? &maps.k : &maps.v);
  if (warp == 1) {
    tmem_alloc(tmem_holder, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_holder;

  if (warp < 4) {
    setmaxnreg_dec<kPtRegsControl>();
    if (warp == 0) {
      // ---------------------------------------------------------- producer
      if (lane == 0) mbar_arrive_expect_tx(q_full, nq * HV * tok * a.G * 128);
      __syncwarp();
      if (lane < nq * HV) {
        const int i = lane / HV, h = lane % HV;
        tma_load_3d(smem + S::Q_OFF + i * S::QTILE + h * kQHalf, &maps.q, q_full, h * 64, hk * a.G,
                    static_cast<int32_t>(rq.t0 + i0 + i * tok));
      }
      const int32_t none = static_cast<int32_t>(a.n_pages * a.Hkv);  // a box outside the pool
      // lane's box of a key tile: its page (or none)
      auto page_of = [&](int u) -> int32_t {
        if (lane >= boxes || u >= u1) return -1;
        const int64_t key = static_cast<int64_t>(all.at(u)) * kTileKeys + lane * box;
        return key < key_end ? __ldg(table + (key >> a.page_shift)) : -1;
      };
      int32_t page = page_of(u0);
      int k_laps = 0, v_laps = 0;
      bool ok = true;
      for (int u = 0; u < nu && ok; ++u) {
        const int st = u % ST;
        const uint32_t ph = (u / ST) & 1u;
        const int kt = all.at(u0 + u);
        const bool have = page >= 0 && page < a.n_pages;
        const int32_t z = have ? page * a.Hkv + hk : none;
        const int32_t y = static_cast<int32_t>((static_cast<int64_t>(kt) * kTileKeys + lane * box) &
                                               ((int64_t{1} << a.page_shift) - 1));
        page = page_of(u0 + u + 1);
        ok = __all_sync(0xffffffffu, mbar_wait(&k_empty[st], ph ^ 1u, status, kDevWaitProducer, abort_flag));
        if (!ok) break;
        if (lane == 0) mbar_arrive_expect_tx(&k_full[st], S::TILE);
        __syncwarp();
        k_laps = u + 1;
        if (lane < boxes)
          for (int h = 0; h < HV; ++h)
            tma_load_3d(smem + S::K_OFF + st * S::TILE + h * kHalf + lane * box * 128, &maps.k, &k_full[st], h * 64, y, z);
        ok = __all_sync(0xffffffffu, mbar_wait(&v_empty[st], ph ^ 1u, status, kDevWaitProducer, abort_flag));
        if (!ok) break;
        if (lane == 0) mbar_arrive_expect_tx(&v_full[st], S::TILE);
        __syncwarp();
        v_laps = u + 1;
        if (lane < boxes)
          for (int h = 0; h < HV; ++h)
            tma_load_3d(smem + S::V_OFF + st * S::TILE + h * kHalf + lane * box * 128, &maps.v, &v_full[st], h * 64, y, z);
      }
      // Every issued copy lands before the CTA may exit: the last lap of each stage.
      mbar_wait(q_full, 0, status, kDevWaitDrain, nullptr);
      for (int u = max(0, k_laps - ST); u < k_laps; ++u)
        mbar_wait(&k_full[u % ST], (u / ST) & 1u, status, kDevWaitDrain, nullptr);
      for (int u = max(0, v_laps - ST); u < v_laps; ++u)
        mbar_wait(&v_full[u % ST], (u / ST) & 1u, status, kDevWaitDrain, nullptr);
    } else if (warp <= 2) {
      // ------------------------------------------- MMAs of query tile warp - 1
      const int i = warp - 1;
      if (i < nq && elect_one()) {
        constexpr uint32_t idesc_qk = idesc_16<BF16>(128, kTileKeys);
        constexpr uint32_t idesc_pv = idesc_16<BF16>(128, D) | (1u << 16);  // B (V) MN-major
        const TileList mine = i == 0 ? own[0] : own[1];
        const uint64_t q_desc = smem_desc_k_sw128(smem_u32(smem + S::Q_OFF + i * S::QTILE));
        const uint64_t k_desc = smem_desc_k_sw128(smem_u32(smem + S::K_OFF));
        const uint64_t v_desc = pt_desc_v(smem_u32(smem + S::V_OFF), HV > 1 ? kHalf : 0);
        const uint32_t s_tmem = tmem + S::S + i * 128, o_tmem = tmem + S::O + i * D;
        bool ok = mbar_wait(q_full, 0, status, kDevWaitMma, abort_flag);
        // Tiles in the order of the rings; of the tile's own ones, S of the next is
        // issued ahead of P V of this one.  A stage that this query tile does not
        // need is released once it has landed.
        int n = 0, prev = -1;  // own tiles so far; number of the previous tile if it is an own one
        bool first = true;
        for (int u = 0; u <= nu && ok; ++u) {
          int x = -1;
          if (u < nu) {
            const int st = u % ST, kt = all.at(u0 + u);
            ok = mbar_wait(&k_full[st], (u / ST) & 1u, status, kDevWaitMma, abort_flag);
            if (!ok) break;
            if (kt < mine.su || (kt >= mine.wu && kt < mine.hu)) {
              x = n++;
              tc_fence_after();
#pragma unroll
              for (int kk = 0; kk < D / 16; ++kk)  // descriptor addresses are in 16-byte units
                mma_f16(s_tmem + (x & 1) * 64, q_desc + ((kk / 4) * kQHalf + (kk % 4) * 32) / 16,
                        k_desc + st * (S::TILE / 16) + ((kk / 4) * kHalf + (kk % 4) * 32) / 16, idesc_qk, kk > 0 ? 1u : 0u);
              mma_commit(&s_full[2 * i + (x & 1)]);
              mma_commit(&k_empty[st]);
            } else {
              mbar_arrive(&k_empty[st]);
            }
          }
          if (u > 0) {
            const int st = (u - 1) % ST;
            ok = mbar_wait(&v_ok[st], ((u - 1) / ST) & 1u, status, kDevWaitMma, abort_flag);
            if (!ok) break;
            if (prev >= 0) {
              ok = mbar_wait(&p_full[2 * i + (prev & 1)], (prev >> 1) & 1u, status, kDevWaitMma, abort_flag);
              if (!ok) break;
              tc_fence_after();
#pragma unroll
              for (int kk = 0; kk < kTileKeys / 16; ++kk)
                mma_f16_ts(o_tmem, s_tmem + (prev & 1) * 64 + kk * 8, v_desc + st * (S::TILE / 16) + kk * (2048 / 16),
                           idesc_pv, (kk > 0 || !first) ? 1u : 0u);
              first = false;
              mma_commit(&pv_full[2 * i + (prev & 1)]);
              mma_commit(&v_empty[st]);
            } else {
              mbar_arrive(&v_empty[st]);
            }
          }
          prev = x;
        }
        if (ok) mma_commit(&o_full[i]);
        mma_commit(&done[i]);
        mbar_wait(&done[i], 0, status, kDevWaitDrain, nullptr);
      }
      __syncwarp();
    } else {
      // ------------------------------------------------- V of the edge tiles
      int edges = 0;
      for (int u = 0; u < nu; ++u) {
        const int st = u % ST, kt = all.at(u0 + u);
        const bool ok = __all_sync(0xffffffffu, mbar_wait(&v_full[st], (u / ST) & 1u, status, kDevWaitEpilogue, abort_flag));
        if (!ok) break;
        if (!plain(kt)) {
          const int64_t k0 = static_cast<int64_t>(kt) * kTileKeys;
          uint8_t* v = smem + S::V_OFF + st * S::TILE;
          const int e = min(edges, kMaxEdges - 1);
          ++edges;
          for (int r = lane; r < kTileKeys; r += 32) {
            const int64_t key = k0 + r;
            const bool some = key < key_end && (a.window <= 0 || key > p_lo - a.window || key < a.sinks);
            bool zero = !some;
            if (some) {
              uint32_t nf = 0;
              for (int x = 0; x < 8 * HV; ++x) {
                const uint4 w = *reinterpret_cast<const uint4*>(v + (x >> 3) * kHalf + r * 128 + ((x + lane) & 7) * 16);
                nf |= nonfinite2<BF16>(w.x) | nonfinite2<BF16>(w.y) | nonfinite2<BF16>(w.z) | nonfinite2<BF16>(w.w);
              }
              if (nf) {
                zero = true;
                bad_kt[e] = static_cast<uint32_t>(kt);  // the same value from every thread
                atomicOr(&bad[e * 4 + (r >> 5)], 1u << (r & 31));
                atomicMax(n_edges, static_cast<uint32_t>(e + 1));
              }
            }
            if (zero)
              for (int x = 0; x < 8 * HV; ++x)
                *reinterpret_cast<uint4*>(v + (x >> 3) * kHalf + r * 128 + ((x + lane) & 7) * 16) = make_uint4(0, 0, 0, 0);
          }
          fence_proxy_async_smem();
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&v_ok[st]);
      }
      asm volatile("bar.sync 1, 288;" ::: "memory");  // the list of bad keys is complete
    }
  } else {
    // ---------------------------------------------------------------- softmax
    setmaxnreg_inc<kPtRegsSoftmax>();
    const int i = (warp - 4) >> 2;   // query tile of this warpgroup
    const int qw = warp & 3;         // TMEM lane quarter
    const int row = qw * 32 + lane;  // row within the tile
    const int64_t t = i0 + static_cast<int64_t>(i) * tok + row / a.G;  // token within the request
    const int64_t h = static_cast<int64_t>(hk) * a.G + row % a.G;
    const bool real = i < nq && row < tok * a.G && t < rq.n;
    const int64_t pos = real ? rq.first + t : kNowhere;
    const uint32_t lane_addr = static_cast<uint32_t>(qw * 32) << 16;
    const uint32_t ts0 = tmem + lane_addr + S::S + i * 128;
    const uint32_t to = tmem + lane_addr + S::O + i * D;
    float m = -INFINITY, l = 0.0f;
    bool ok = true;
    const int jb = i == 0 ? j0[0] : j0[1], je = i == 0 ? j1[0] : j1[1];
    const TileList mine = i == 0 ? own[0] : own[1];
    // Which pages of a tile exist is asked tile by tile only if one of the stretch's is
    // absent (a table read and a vote in every tile cost a tenth of it).
    auto entry = [&](int kt) -> int32_t {  // lane's page of tile kt (present where there is none to ask for)
      const int64_t key = static_cast<int64_t>(kt) * kTileKeys + lane * box;
      return lane < boxes && key < rq.len ? __ldg(table + (key >> a.page_shift)) : 0;
    };
    bool holes = false;
    if (jb < je) {
      const int last = mine.at(je - 1);
      auto scan = [&](int from, int to) {  // tiles from .. to
        const int64_t e0 = (static_cast<int64_t>(from) * kTileKeys) >> a.page_shift;
        const int64_t e1 = min(static_cast<int64_t>(to) * kTileKeys + kTileKeys - 1, rq.len - 1) >> a.page_shift;
        for (int64_t e = e0 + lane; e <= e1; e += 32) {
          const int32_t pg = __ldg(table + e);
          holes |= pg < 0 || pg >= a.n_pages;
        }
      };
      if (jb < mine.su) scan(mine.at(jb), min(last, mine.su - 1));
      if (je > mine.su) scan(mine.at(max(jb, mine.su)), last);
      holes = __any_sync(0xffffffffu, holes);
    }
    // tiles below plain_hi, at or past plain_lo or below plain_sk, are seen whole by every row
    const int plain_hi = static_cast<int>(max(int64_t{0}, (a.causal ? min(rq.len, p_lo + 1) : rq.len)) / kTileKeys);
    const int plain_lo =
        a.window > 0 ? static_cast<int>((max(int64_t{0}, p_hi - a.window + 1) + kTileKeys - 1) / kTileKeys) : 0;
    const int plain_sk = static_cast<int>(a.window > 0 ? min(a.sinks, rq.len) / kTileKeys : 0);
    const int row_bit = min(a.page_shift, 6);
    const bool positive = a.c2 > 0.0f;
    const float cc = positive ? a.c2 : 1.0f;  // scores times this are in powers of two
    for (int j = jb; j < je; ++j) {
      const int x01 = (j - jb) & 1;
      const uint32_t par = ((j - jb) >> 1) & 1u, ts = ts0 + x01 * 64;
      if (!__all_sync(0xffffffffu, mbar_try_wait(&s_full[2 * i + x01], par)))
        ok = __all_sync(0xffffffffu, mbar_wait(&s_full[2 * i + x01], par, status, kDevWaitEpilogue, abort_flag));
      if (!ok) break;
      tc_fence_after();
      uint32_t sr[kTileKeys];
#pragma unroll
      for (int x = 0; x < kTileKeys; x += 32) tmem_ld_32x32b_x32(ts + x, *reinterpret_cast<uint32_t(*)[32]>(&sr[x]));
      tmem_wait_ld();
      if (!positive) {  // rare: the order of the scaled scores is another one (before the masks: -inf is a score too)
#pragma unroll
        for (int x = 0; x < kTileKeys; ++x) sr[x] = __float_as_uint(__uint_as_float(sr[x]) * a.c2);
      }
      const int kt = mine.at(j);
      if (holes || kt >= plain_hi || (kt < plain_lo && kt >= plain_sk)) {
        uint32_t pages = 0xffffffffu;
        if (holes) {
          const int32_t pg = entry(kt);
          pages = __ballot_sync(0xffffffffu, pg >= 0 && pg < a.n_pages);
        }
        const int64_t k0 = static_cast<int64_t>(kt) * kTileKeys;
        // visible: x < hi and (x >= lo or x < sk), page present
        const int64_t hi64 = (a.causal ? min(rq.len, pos + 1) : (real ? rq.len : 0)) - k0;
        const int64_t lo64 = a.window > 0 ? pos - a.window + 1 - k0 : 0;
        const int64_t sk64 = a.window > 0 ? a.sinks - k0 : 0;
        const int hi = static_cast<int>(max(int64_t{-1}, min(hi64, int64_t{kTileKeys})));
        const int lo = static_cast<int>(max(int64_t{-1}, min(lo64, int64_t{kTileKeys})));
        const int sk = static_cast<int>(max(int64_t{-1}, min(sk64, int64_t{kTileKeys})));
#pragma unroll
        for (int x = 0; x < kTileKeys; ++x)
          if (!(x < hi && (x >= lo || x < sk) && ((pages >> (x >> row_bit)) & 1u))) sr[x] = __float_as_uint(-INFINITY);
      }
      float mx8[8];  // row max: three-input max, eight chains
#pragma unroll
      for (int x = 0; x < 8; ++x) mx8[x] = __uint_as_float(sr[x]);
#pragma unroll
      for (int x = 8; x < kTileKeys; x += 16)
#pragma unroll
        for (int y = 0; y < 8; ++y)
          mx8[y] = pt_max3(mx8[y], __uint_as_float(sr[x + y]), x + 8 + y < kTileKeys ? __uint_as_float(sr[x + 8 + y]) : mx8[y]);
      const float mx = cc * pt_max3(pt_max3(mx8[0], mx8[1], mx8[2]), pt_max3(mx8[3], mx8[4], mx8[5]), pt_max3(mx8[6], mx8[7], mx8[7]));
      if (!(mx < INFINITY)) l = NAN;  // a NaN or an infinite score: the row is NaN, whatever its exps give
      float m_new = fmaxf(m, mx);
      const bool grow = m_new > m + 8.0f || (m == -INFINITY && m_new != -INFINITY);
      if (!grow) m_new = m;
      const float base = m_new == -INFINITY ? 0.0f : m_new;
      const float alpha = !grow || m == -INFINITY ? (grow ? 0.0f : 1.0f) : ex2(m - m_new);
      uint32_t pk[kTileKeys / 2];
      {
        const float2 nm = make_float2(-base, -base), one = make_float2(1.0f, 1.0f), c2 = make_float2(cc, cc);
        float2 ls[4] = {make_float2(0.0f, 0.0f), make_float2(0.0f, 0.0f), make_float2(0.0f, 0.0f), make_float2(0.0f, 0.0f)};
#pragma unroll
        for (int x = 0; x < kTileKeys; x += 2) {
          const float2 z = ffma2(make_float2(__uint_as_float(sr[x]), __uint_as_float(sr[x + 1])), c2, nm);
          const float2 y = ((x >> 1) & 3) < kPolyPairs ? pt_ex2_poly(z) : make_float2(ex2(z.x), ex2(z.y));
          pk[x >> 1] = pack2<BF16>(y.x, y.y);
          ls[(x >> 1) & 3] = ffma2(y, one, ls[(x >> 1) & 3]);
        }
        l = fmaf(l, alpha, ((ls[0].x + ls[0].y) + (ls[1].x + ls[1].y)) + ((ls[2].x + ls[2].y) + (ls[3].x + ls[3].y)));
      }
      if (j > jb && __any_sync(0xffffffffu, grow)) {
        // Rescale O, once the previous P V is in it.  Its barrier can be in that phase or
        // just past it: the P V two before that came ahead of a score tile already read,
        // the next one waits for this warp.
        const int prev = j - jb - 1;
        ok = __all_sync(0xffffffffu, mbar_wait(&pv_full[2 * i + (prev & 1)], (prev >> 1) & 1u, status, kDevWaitEpilogue, abort_flag));
        if (!ok) break;
        tc_fence_after();
#pragma unroll
        for (int d = 0; d < D; d += 32) {
          uint32_t r[32];
          tmem_ld_32x32b_x32(to + d, r);
          tmem_wait_ld();
#pragma unroll
          for (int x = 0; x < 32; ++x) r[x] = __float_as_uint(__uint_as_float(r[x]) * alpha);
          tmem_st_32x32b_x32(to + d, r);
        }
      }
      tmem_st_32x32b_x32(ts, pk);
      tmem_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&p_full[2 * i + x01]);
      m = m_new;
    }
    if (ok && je > jb)
      ok = __all_sync(0xffffffffu, mbar_wait(&o_full[i], 0, status, kDevWaitEpilogue, abort_flag));
    asm volatile("bar.sync 1, 288;" ::: "memory");  // the list of bad keys is complete
    tc_fence_after();
    if (ok && i < nq) {
      const int64_t tr = rq.t0 + t;
      const bool whole_keys = a.splits == 1;
      const bool empty = m == -INFINITY && l == 0.0f;
      const float inv = whole_keys ? (empty ? 0.0f : 1.0f / l) : 1.0f;
      const int64_t pi = (tr * a.Hq + h) * a.splits + split;
      if (real && !whole_keys) a.part_ml[pi] = make_float2(m, l);
      const int n_bad = static_cast<int>(*reinterpret_cast<volatile uint32_t*>(n_edges));
      for (int d = 0; d < D; d += 32) {
        uint32_t r[32];
        if (je > jb) {
          tmem_ld_32x32b_x32(to + d, r);
          tmem_wait_ld();
        } else {
#pragma unroll
          for (int x = 0; x < 32; ++x) r[x] = 0u;
        }
        if (real) {
        float o[32];
#pragma unroll
        for (int x = 0; x < 32; ++x) o[x] = empty ? 0.0f : __uint_as_float(r[x]);
        if (n_bad > 0 && !empty) {  // rare: the shares of keys with non-finite values
          const uint16_t* qr = static_cast<const uint16_t*>(a.q) + tr * a.ldq + h * D;
          for (int e = 0; e < n_bad; ++e)
            for (int w = 0; w < 4; ++w)
              for (uint32_t bits = bad[e * 4 + w]; bits; bits &= bits - 1) {
                const int64_t key = static_cast<int64_t>(bad_kt[e]) * kTileKeys + w * 32 + (__ffs(bits) - 1);
                if (!sees(a, pos, key, rq.len)) continue;
                const int32_t pg = __ldg(table + (key >> a.page_shift));
                if (pg < 0 || pg >= a.n_pages) continue;
                const int64_t off = (((static_cast<int64_t>(pg) * a.Hkv + hk) << a.page_shift) +
                                     (key & ((int64_t{1} << a.page_shift) - 1))) * D;
                float s = 0.0f;
                for (int x = 0; x < D; x += 2) {
                  const float2 qv = unpack2<BF16>(*reinterpret_cast<const uint32_t*>(qr + x));
                  const float2 kv = unpack2<BF16>(*reinterpret_cast<const uint32_t*>(a.k + off + x));
                  s = fmaf(qv.x, kv.x, fmaf(qv.y, kv.y, s));
                }
                const float p = exp2f(s * a.c2 - m);
#pragma unroll
                for (int x = 0; x < 32; x += 2) {
                  const float2 vv = unpack2<BF16>(*reinterpret_cast<const uint32_t*>(a.v + off + d + x));
                  o[x] = fmaf(p, vv.x, o[x]);
                  o[x + 1] = fmaf(p, vv.y, o[x + 1]);
                }
              }
        }
        if (l == l) {  // (an empty row is 0 by now)
          bool lost = false;
#pragma unroll
          for (int x = 0; x < 32; ++x) lost |= o[x] != o[x];
          if (lost) {  // an infinite value met a weight of 0
            const int hi = static_cast<int>(max(int64_t{0}, a.causal ? min(rq.len, pos + 1) : rq.len));
            const int lo = a.window > 0 ? static_cast<int>(max(int64_t{0}, pos - a.window + 1)) : 0;
            const uint2 seen = nonfinite_seen<16, BF16>(
                a.v + ((static_cast<int64_t>(hk) * D) << a.page_shift) + d, table, a.n_pages, a.page_shift,
                (static_cast<int64_t>(a.Hkv) * D) << a.page_shift, D, lo, hi, a.window > 0 ? static_cast<int>(a.sinks) : 0);
#pragma unroll
            for (int x = 0; x < 32; ++x)
              if (o[x] != o[x]) o[x] = settled(seen, x);
          }
        }
        if (whole_keys) {
          uint16_t* dst = static_cast<uint16_t*>(a.o) + tr * a.ldo + h * D + d;
#pragma unroll
          for (int x = 0; x < 32; x += 8) {
            uint4 w;
            w.x = pack2<BF16>(o[x] * inv, o[x + 1] * inv);
            w.y = pack2<BF16>(o[x + 2] * inv, o[x + 3] * inv);
            w.z = pack2<BF16>(o[x + 4] * inv, o[x + 5] * inv);
            w.w = pack2<BF16>(o[x + 6] * inv, o[x + 7] * inv);
            *reinterpret_cast<uint4*>(dst + x) = w;
          }
        } else {
          float* dst = a.part_o + pi * D + d;
#pragma unroll
          for (int x = 0; x < 32; x += 4)
            *reinterpret_cast<float4*>(dst + x) = make_float4(o[x], o[x + 1], o[x + 2], o[x + 3]);
        }
        }
        __syncwarp();
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

template <int D, bool BF16>
cudaError_t launch_tiles(const PagedArgs& a, cudaStream_t s) {
  using S = PtShape<D>;
  static_assert(S::BYTES <= 227 * 1024, "shared memory");
  const int tok = kTileRows / a.G;
  PtMaps maps;
  const CUtensorMapDataType dt = BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  const uint64_t page = uint64_t{1} << a.page_shift;
  const uint64_t qd[3] = {D, static_cast<uint64_t>(a.Hq), static_cast<uint64_t>(a.T)};
  const uint64_t qs[2] = {D * 2, static_cast<uint64_t>(a.ldq) * 2};
  const uint32_t qb[3] = {64, static_cast<uint32_t>(a.G), static_cast<uint32_t>(tok)};
  const uint64_t kd[3] = {D, page, static_cast<uint64_t>(a.n_pages) * a.Hkv};
  const uint64_t ks[2] = {D * 2, page * D * 2};
  const uint32_t kb[3] = {64, static_cast<uint32_t>(page < kTileKeys ? page : kTileKeys), 1};
  if (!make_tensor_map_3d(&maps.q, dt, a.q, qd, qs, qb, CU_TENSOR_MAP_SWIZZLE_128B) ||
      !make_tensor_map_3d(&maps.k, dt, a.k, kd, ks, kb, CU_TENSOR_MAP_SWIZZLE_128B) ||
      !make_tensor_map_3d(&maps.v, dt, a.v, kd, ks, kb, CU_TENSOR_MAP_SWIZZLE_128B))
    return cudaErrorInvalidValue;
  auto kern = paged_tile_kernel<D, BF16>;
  static bool attr_set[64] = {};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return cudaErrorInvalidDevice;
  if (!attr_set[dev]) {
    // The register split needs the kernel compiled at exactly kPtLaunchRegs, or
    // setmaxnreg.inc could wait for registers that do not exist.
    cudaFuncAttributes fa;
    cudaError_t e = cudaFuncGetAttributes(&fa, kern);
    if (e != cudaSuccess) return e;
    if (fa.numRegs != kPtLaunchRegs) return cudaErrorInvalidConfiguration;
    e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, S::BYTES);
    if (e != cudaSuccess) return e;
    attr_set[dev] = true;
  }
  const int64_t tiles = (a.max_q + 2 * tok - 1) / (2 * tok);
  if (tiles * a.splits > INT32_MAX) return cudaErrorInvalidValue;
  const dim3 grid(static_cast<unsigned>(tiles * a.splits), static_cast<unsigned>(a.Hkv), static_cast<unsigned>(a.B));
  kern<<<grid, kPtThreads, S::BYTES, s>>>(maps, a, tok);
  const cudaError_t e = cudaGetLastError();
  return e != cudaSuccess || a.splits == 1 ? e : launch_paged_join(a, D, BF16, s);
}

}  // namespace

cudaError_t launch_paged_tiles(const PagedArgs& a, int D, bool bf16, cudaStream_t s) {
  if (D == 64) return bf16 ? launch_tiles<64, true>(a, s) : launch_tiles<64, false>(a, s);
  return bf16 ? launch_tiles<128, true>(a, s) : launch_tiles<128, false>(a, s);
}

cudaError_t read_paged_status(unsigned int* value, bool clear) {
  cudaError_t e = cudaMemcpyFromSymbol(value, g_paged_status, sizeof(unsigned int));
  if (e != cudaSuccess || !clear) return e;
  const unsigned int zero = 0;
  return cudaMemcpyToSymbol(g_paged_status, &zero, sizeof(unsigned int));
}

}  // namespace b2q
