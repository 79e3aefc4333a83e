// b2q_attention_paged.cu -- attention of each request's newest tokens over its
// keys and values in a paged cache, ragged over requests, grouped heads.
//
//   cache [page][kv head][token in page][D], 16-bit; page ids in table[b][.]
//   token i of the n new ones of a request of length L sits at p = L - n + i;
//   it sees key j when j < L, j's page is present, j <= p (causal) and, with a
//   window w, j > p - w or j < sinks
//   o = sum_j e_j v_j / sum_j e_j,  e_j = 2^((q . k_j) scale log2(e) - max),
//   a row that sees nothing is 0
//
// The rows of one kv head are its (token, query head of the group) pairs, token
// major: a key is read once for all of them.
//
// Few rows (paged_rows_kernel): bound by the cache's bytes.  A CTA of four
// warps takes 16 rows, or 32 (RT 2), and one stretch of the keys.  With 16 rows
// every warp takes units of 16 keys in turn, with a ring of cp.async stages of its
// own (no barrier inside the loop), its own running maxima, sums and outputs, and
// they join at the end.  With 32, two warps share a ring, each copies half of a
// unit and works on 16 of the rows, and a barrier of the two stands where a warp
// alone has none.  (Two CTAs of 16 rows instead read the keys twice, and the L2 did
// not make up for it: 24 rows over 120k keys took 192 us.)  A unit lies inside one
// page (pages are multiples of 16), keys that no row of the CTA sees are not loaded
// but filled with zeros.  Products are m16n8k16; P is fed to the second product as
// two 16-bit numbers, P and what rounding it left: the tensor pipe idles behind the
// loads, and a single rounding of P would cost as much accuracy as the output's own.
// Stretches are split over CTAs when the rows alone do not fill the GPU; a
// second kernel then joins their outputs by their maxima and sums.
// Measured (32 / 8 heads of 128): 64 requests of 0.9k to 24k keys 480 us,
// 6800 GB/s; one of 120k keys 85 us, 5800 GB/s; 3 requests of 16 heads of 64
// over at most 900 keys 10.5 us, two launches and one CTA's chain of units.
#include "b2q_internal.h"
#include "b2q_paged.cuh"
#include "b2q_ptx.cuh"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cmath>

namespace b2q {

namespace {

constexpr int kRowsWarps = 4;
constexpr int kRowsThreads = kRowsWarps * 32;
constexpr int kUnit = 16;  // keys

template <bool BF16>
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (BF16) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  } else {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
}
__device__ __forceinline__ void ldsm4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldsm4_t(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
// 16 bytes to shared memory, or 16 zero bytes (nothing is read then).
__device__ __forceinline__ void cp16(uint32_t dst, const void* src, bool real) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(real ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
template <int D, int RT>
struct RowsShape {
  static constexpr int GROUPS = kRowsWarps / RT;         // of RT warps with a ring each
  static constexpr int STAGES = RT == 1 ? (D == 64 ? 4 : 3) : (D == 64 ? 8 : 4);
  static constexpr int KV = kUnit * D * 2;               // bytes of one unit's keys (or values)
  static constexpr int RING = STAGES * 2 * KV;           // per group
  static constexpr int BYTES = GROUPS * RING;
};

template <int D, bool BF16, int RT>
__global__ void __launch_bounds__(kRowsThreads) paged_rows_kernel(const PagedArgs a, const int tiles) {
  using S = RowsShape<D, RT>;
  constexpr int CH = D / 8;         // 16-byte chunks of a row
  constexpr int RPI = 32 / CH;      // rows that a warp copies at a time
  constexpr int COPIES = kUnit / RT / RPI;
  constexpr int ROWS = 16 * RT;     // of the CTA
  extern __shared__ __align__(128) uint8_t rows_smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int group = warp / RT, rt = warp % RT;
  const int b = blockIdx.z, hk = blockIdx.y;
  const int split = blockIdx.x / tiles, tile = blockIdx.x % tiles;
  const Request rq = request_of(a, b);
  const int64_t rows = rq.n * a.G;
  const int64_t r0 = static_cast<int64_t>(tile) * ROWS;
  if (r0 >= rows) return;
  const int64_t p_lo = rq.first + r0 / a.G, p_hi = rq.first + min(rows - 1, r0 + ROWS - 1) / a.G;
  const Units un = units_of(a, rq.len, p_lo, p_hi, kUnit);
  // the last stretch takes what a longer request than announced has left
  const int u_all = static_cast<int>(un.count());
  const int u0 = static_cast<int>(min(static_cast<int64_t>(split) * a.split_units, static_cast<int64_t>(u_all)));
  const int u1 =
      split == a.splits - 1 ? u_all : static_cast<int>(min(static_cast<int64_t>(u_all), u0 + a.split_units));
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");  // the joining kernel may get ready
  if (split > 0 && u0 >= u_all) {  // no keys in this stretch
    const int64_t r = r0 + threadIdx.x;
    if (threadIdx.x < ROWS && r < rows)
      a.part_ml[((rq.t0 + r / a.G) * a.Hq + static_cast<int64_t>(hk) * a.G + r % a.G) * a.splits + split] =
          make_float2(-INFINITY, 0.0f);
    return;
  }
  const int su = static_cast<int>(un.su), gap = static_cast<int>(un.wu - un.su);
  auto unit_at = [&](int i) { return i < su ? i : i + gap; };

  // Keys: rows of the CTA see [win_lo, key_end) and [0, sinks); every one sees
  // [full_lo, full_hi) and the sinks below full_hi.
  const int key_end = static_cast<int>(max(int64_t{0}, a.causal ? min(rq.len, p_hi + 1) : rq.len));
  const int win_lo = static_cast<int>(un.win_lo);
  const int full_hi = static_cast<int>(max(int64_t{0}, a.causal ? min(rq.len, p_lo + 1) : rq.len));
  const int full_lo = a.window > 0 ? static_cast<int>(max(int64_t{0}, p_hi - a.window + 1)) : 0;
  const int sinks = a.window > 0 ? static_cast<int>(a.sinks) : 0;

  // Rows of this thread: g and g + 8 of its warp's 16; each sees [lo, hi) and the sinks below hi.
  const int g = lane >> 2, c = lane & 3;
  int lo[2], hi[2];
  uint32_t qf[D / 16][4];
  const uint16_t* qp = static_cast<const uint16_t*>(a.q);
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const int64_t r = r0 + rt * 16 + g + 8 * e;
    const bool real = r < rows;
    const int64_t i = real ? r / a.G : 0, pos = rq.first + i;
    hi[e] = real ? static_cast<int>(max(int64_t{0}, a.causal ? min(rq.len, pos + 1) : rq.len)) : 0;
    lo[e] = a.window > 0 ? static_cast<int>(max(int64_t{0}, pos - a.window + 1)) : 0;
    const uint16_t* src = qp + (rq.t0 + i) * a.ldq + (static_cast<int64_t>(hk) * a.G + (real ? r % a.G : 0)) * D;
#pragma unroll
    for (int ks = 0; ks < D / 16; ++ks) {
      qf[ks][e] = real ? *reinterpret_cast<const uint32_t*>(src + ks * 16 + 2 * c) : 0u;
      qf[ks][2 + e] = real ? *reinterpret_cast<const uint32_t*>(src + ks * 16 + 8 + 2 * c) : 0u;
    }
  }

  float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f}, o[D / 8][4];
#pragma unroll
  for (int j = 0; j < D / 8; ++j) o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.0f;

  const bool idle = r0 + rt * 16 >= rows;  // copies its half, and has no row of its own
  auto together = [&] {  // the warps of a ring
    if constexpr (RT == 1)
      __syncwarp();
    else
      asm volatile("bar.sync %0, %1;" ::"r"(1 + group), "n"(32 * RT) : "memory");
  };
  uint8_t* ring = rows_smem + group * S::RING;
  const uint32_t ring_a = smem_u32(ring);
  const int32_t* table = a.table + static_cast<int64_t>(b) * a.ldt;
  const int64_t page_elems = static_cast<int64_t>(a.Hkv) * D << a.page_shift;
  const int64_t lane_elems = (static_cast<int64_t>(hk) * D << a.page_shift) + rt * (kUnit / RT) * D + lane * 8;
  const int page_mask = (1 << a.page_shift) - 1;
  // Chunk ch of row r sits at chunk ch ^ (r % 8) of its 128 bytes.  A lane copies
  // chunk lane % CH of rows lane / CH + RPI x of its warp's share; reads keys (lane & 7) + 8 (lane / 16)
  // of K, (lane & 7) + 8 (lane / 8 % 2) of V.
  const int cr = rt * (kUnit / RT) + lane / CH, cc = lane % CH;
  uint32_t cp_off[COPIES < 4 ? COPIES : 4];
#pragma unroll
  for (int x = 0; x < (COPIES < 4 ? COPIES : 4); ++x) {
    const int r = cr + RPI * x;
    cp_off[x] = r * (D * 2) + ((cc & ~7) | ((cc ^ r) & 7)) * 16;
  }
  const int krow = (lane & 7) + ((lane >> 4) << 3), vrow = (lane & 7) + (((lane >> 3) & 1) << 3);
  const uint32_t k_off = krow * (D * 2) + ((((lane >> 3) & 1) ^ krow) & 7) * 16;
  const uint32_t v_off = vrow * (D * 2) + (((lane >> 4) ^ vrow) & 7) * 16;

  uint32_t present = 0;  // bit s: stage s holds a page's keys
  // The page of unit i of the stretch (-1: none).
  auto page_of = [&](int i) -> int32_t {
    return i < u1 ? __ldg(table + ((unit_at(i) * kUnit) >> a.page_shift)) : -1;
  };
  auto load = [&](int i, int stage, int32_t page) {
    present &= ~(1u << stage);
    if (i < u1) {
      const int k0 = unit_at(i) * kUnit;
      const bool have = page >= 0 && page < a.n_pages;
      const int64_t off = (have ? static_cast<int64_t>(page) * page_elems : 0) + lane_elems + (k0 & page_mask) * D;
      const uint32_t kd = ring_a + stage * 2 * S::KV;
      if (have) present |= 1u << stage;
      if (have && k0 + kUnit <= key_end && (k0 >= win_lo || k0 + kUnit <= sinks)) {
#pragma unroll
        for (int x = 0; x < COPIES; ++x) {
          const uint32_t d = kd + cp_off[x & 3] + (x >> 2) * 4 * RPI * (D * 2);
          cp16(d, a.k + off + x * 256, true);
          cp16(d + S::KV, a.v + off + x * 256, true);
        }
      } else {
#pragma unroll
        for (int x = 0; x < COPIES; ++x) {
          const int key = k0 + cr + RPI * x;
          const bool real = have && key < key_end && (key >= win_lo || key < sinks);
          const uint32_t d = kd + cp_off[x & 3] + (x >> 2) * 4 * RPI * (D * 2);
          cp16(d, real ? a.k + off + x * 256 : a.k, real);
          cp16(d + S::KV, real ? a.v + off + x * 256 : a.v, real);
        }
      }
    }
    cp_commit();  // an empty group keeps the count
  };

  // Ring: the group's units are u0 + group, + GROUPS, ..
  int next = u0 + group;
#pragma unroll
  for (int s = 0; s < S::STAGES - 1; ++s, next += S::GROUPS) load(next, s, page_of(next));
  int32_t next_page = page_of(next);
  int stage = 0, fill = S::STAGES - 1;
  for (int i = u0 + group; i < u1; i += S::GROUPS) {
    cp_wait<S::STAGES - 2>();
    together();  // the unit is there, and the stage before it has been read by all
    const uint32_t ka = ring_a + stage * 2 * S::KV, va = ka + S::KV;
    const int k0 = unit_at(i) * kUnit;

    const bool page_in = (present >> stage) & 1u;
    const bool full = page_in && k0 + kUnit <= full_hi && (k0 >= full_lo || k0 + kUnit <= sinks);
    const bool mixed = !full && page_in && p_lo < p_hi;
    auto refill = [&] {  // the stage before this one
      const int32_t pg = next_page;
      next_page = page_of(next + S::GROUPS);
      load(next, fill, pg);
      next += S::GROUPS;
    };
    if (RT > 1 && idle && !mixed) {
      refill();
      stage = stage + 1 == S::STAGES ? 0 : stage + 1;
      fill = fill + 1 == S::STAGES ? 0 : fill + 1;
      continue;
    }
    float s[2][2][4];  // two accumulation chains per 8 keys
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int x = 0; x < 4; ++x) s[0][t][x] = s[1][t][x] = 0.0f;
#pragma unroll
    for (int ks = 0; ks < D / 16; ++ks) {
      uint32_t kf[4];
      ldsm4(((ka + k_off) ^ ((ks & 3) * 32)) + (ks >> 2) * 128, kf);
      mma16816<BF16>(s[ks & 1][0], qf[ks], kf[0], kf[1]);
      mma16816<BF16>(s[ks & 1][1], qf[ks], kf[2], kf[3]);
    }
    refill();  // (its instructions fill the time that the products take)
    float mx[2];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int x = 0; x < 2; ++x) s[0][t][2 * e + x] = (s[0][t][2 * e + x] + s[1][t][2 * e + x]) * a.c2;
      if (!full) {
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            const int j = k0 + t * 8 + 2 * c + x;
            if (!(page_in && j < hi[e] && (j >= lo[e] || j < sinks))) s[0][t][2 * e + x] = -INFINITY;
          }
      }
      float v = fmaxf(fmaxf(s[0][0][2 * e], s[0][0][2 * e + 1]), fmaxf(s[0][1][2 * e], s[0][1][2 * e + 1]));
      v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 1));
      v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 2));
      mx[e] = v;
    }
    // The maximum in use is raised only when a unit exceeds it by 2^8: P stays
    // below 2^8, which 16-bit floats hold as exactly as values below 1.
    const bool grow = mx[0] > m[0] + 8.0f || (m[0] == -INFINITY && mx[0] != -INFINITY) || mx[1] > m[1] + 8.0f ||
                      (m[1] == -INFINITY && mx[1] != -INFINITY);
    if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const float nm = fmaxf(m[e], mx[e]);
        const float al = m[e] == -INFINITY ? 0.0f : ex2(m[e] - nm);
        m[e] = nm;
        l[e] *= al;
#pragma unroll
        for (int j = 0; j < D / 8; ++j) {
          o[j][2 * e] *= al;
          o[j][2 * e + 1] *= al;
        }
      }
    }
    uint32_t ph[4], pl[4];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const float base = m[e] == -INFINITY ? 0.0f : m[e];
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        float& x = s[0][t][2 * e];
        float& y = s[0][t][2 * e + 1];
        x = ex2(x - base);
        y = ex2(y - base);
        l[e] += x + y;
        const uint32_t h2 = pack2<BF16>(x, y);
        const float2 h = unpack2<BF16>(h2);
        ph[2 * t + e] = h2;
        pl[2 * t + e] = pack2<BF16>(x - h.x, y - h.y);
      }
    }
    if (mixed) {
      // Rows of this unit see different keys.  A key that some row does not see
      // may hold an infinity or a NaN, and 0 times that is no 0: such keys leave
      // the tensor product (their values are zeroed in the stage) and are added
      // to the rows that see them one by one.
      uint8_t* vs = ring + stage * 2 * S::KV + S::KV;
      uint32_t bad = 0;
#pragma unroll
      for (int x = 0; x < kUnit / RPI; ++x) {
        const uint4 u = *reinterpret_cast<const uint4*>(vs + (lane + 32 * x) * 16);
        if (nonfinite2<BF16>(u.x) || nonfinite2<BF16>(u.y) || nonfinite2<BF16>(u.z) || nonfinite2<BF16>(u.w))
          bad |= 1u << (lane / CH + RPI * x);
      }
      bad = __reduce_or_sync(0xffffffffu, bad);
      if (RT > 1) together();  // all have looked
      for (uint32_t left = bad; left; left &= left - 1) {
        const int r = __ffs(left) - 1, j = k0 + r;
        const int src = (lane & ~3) | ((r & 7) >> 1);
        const uint8_t* vr = vs + r * (D * 2);
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float q0 = __shfl_sync(0xffffffffu, r < 8 ? s[0][0][2 * e] : s[0][1][2 * e], src);
          const float q1 = __shfl_sync(0xffffffffu, r < 8 ? s[0][0][2 * e + 1] : s[0][1][2 * e + 1], src);
          const float p = (r & 1) ? q1 : q0;
          if (j < hi[e] && (j >= lo[e] || j < sinks)) {
#pragma unroll
            for (int d = 0; d < D / 8; ++d) {
              const float2 v =
                  unpack2<BF16>(*reinterpret_cast<const uint32_t*>(vr + ((d & ~7) | ((d ^ r) & 7)) * 16 + c * 4));
              o[d][2 * e] = fmaf(p, v.x, o[d][2 * e]);
              o[d][2 * e + 1] = fmaf(p, v.y, o[d][2 * e + 1]);
            }
          }
        }
      }
      if (bad) {
        together();  // all have added
        for (uint32_t left = bad; left; left &= left - 1)
          if (lane < CH && rt == 0)
            *reinterpret_cast<uint4*>(vs + (__ffs(left) - 1) * (D * 2) + lane * 16) = make_uint4(0, 0, 0, 0);
        together();
      }
    }
#pragma unroll
    for (int j = 0; j < D / 16; ++j) {
      uint32_t vf[4];
      ldsm4_t(((va + v_off) ^ ((j & 3) * 32)) + (j >> 2) * 128, vf);
      mma16816<BF16>(o[2 * j], ph, vf[0], vf[1]);
      mma16816<BF16>(o[2 * j + 1], ph, vf[2], vf[3]);
      mma16816<BF16>(o[2 * j], pl, vf[0], vf[1]);
      mma16816<BF16>(o[2 * j + 1], pl, vf[2], vf[3]);
    }
    if (RT == 1) __syncwarp();  // every lane has read the stage before it is refilled
    stage = stage + 1 == S::STAGES ? 0 : stage + 1;
    fill = fill + 1 == S::STAGES ? 0 : fill + 1;
  }
  cp_wait<0>();
  __syncthreads();

  // Join the four warps: [warp][row] (max, sum), then [warp][row][D].
  float2* ml = reinterpret_cast<float2*>(rows_smem);
  float* ow = reinterpret_cast<float*>(rows_smem) + kRowsWarps * 16 * 2;
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    float v = l[e];
    v += __shfl_xor_sync(0xffffffffu, v, 1);
    v += __shfl_xor_sync(0xffffffffu, v, 2);
    const int row = g + 8 * e;
    if (c == 0) ml[warp * 16 + row] = make_float2(m[e], v);
#pragma unroll
    for (int j = 0; j < D / 8; ++j)
      *reinterpret_cast<float2*>(ow + (warp * 16 + row) * D + j * 8 + 2 * c) = make_float2(o[j][2 * e], o[j][2 * e + 1]);
  }
  __syncthreads();
  constexpr int TPR = kRowsThreads / ROWS;  // threads per row
  const int part = threadIdx.x % TPR, row = threadIdx.x / TPR % 16, own = threadIdx.x / TPR / 16;  // row of tile `own`
  const int64_t r = r0 + own * 16 + row;
  if (r >= rows) return;
  float M = -INFINITY;
#pragma unroll
  for (int w = 0; w < S::GROUPS; ++w) M = fmaxf(M, ml[(w * RT + own) * 16 + row].x);
  float f[S::GROUPS], sum = 0.0f;
#pragma unroll
  for (int w = 0; w < S::GROUPS; ++w) {
    const float2 x = ml[(w * RT + own) * 16 + row];
    f[w] = x.x == -INFINITY ? x.y * 0.0f : ex2(x.x - M);  // (no finite score: 0, or NaN where one was NaN)
    sum += f[w] * x.y;
  }
  const int64_t t = rq.t0 + r / a.G;
  const int64_t h = static_cast<int64_t>(hk) * a.G + r % a.G;
  const bool whole = a.splits == 1;
  const bool empty = M == -INFINITY && sum == 0.0f;
  const float inv = whole ? (empty ? 0.0f : 1.0f / sum) : 1.0f;
  const int64_t pi = (t * a.Hq + h) * a.splits + split;
  if (!whole && part == 0) a.part_ml[pi] = make_float2(M, sum);
#pragma unroll
  for (int d = part * 2; d < D; d += TPR * 2) {
    float x = 0.0f, y = 0.0f;
    if (!empty) {
#pragma unroll
      for (int w = 0; w < S::GROUPS; ++w) {
        const float2 v = *reinterpret_cast<const float2*>(ow + ((w * RT + own) * 16 + row) * D + d);
        if (f[w] != 0.0f) {  // a warp without keys adds nothing, whatever it holds
          x = fmaf(f[w], v.x, x);
          y = fmaf(f[w], v.y, y);
        }
      }
    }
    if (whole)
      *reinterpret_cast<uint32_t*>(static_cast<uint16_t*>(a.o) + t * a.ldo + h * D + d) = pack2<BF16>(x * inv, y * inv);
    else
      *reinterpret_cast<float2*>(a.part_o + pi * D + d) = make_float2(x, y);
  }
}

// o = sum_s 2^(m_s - M) O_s / sum_s 2^(m_s - M) l_s over the splits, in their
// order, for one (token, query head) a CTA.  The splits' weights are worked out
// once, side by side; then every thread adds up its values, loads ahead.  Launched
// with the attention kernel still running (it waits before it reads): 94 -> 83 us
// for one request of 120k keys, with the warp-wide loop over 37 splits before.
constexpr int kJoinMax = 1024;  // splits

template <int D, bool BF16>
__global__ void __launch_bounds__(D / 2) paged_join_kernel(const PagedArgs a) {
  __shared__ float f[kJoinMax];
  __shared__ float red[2][D / 64];
  const int tid = threadIdx.x, lane = tid & 31;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const Request rq = request_of(a, blockIdx.y);
  const int i = blockIdx.x / a.Hq, h = blockIdx.x - i * a.Hq;
  if (i >= rq.n) return;
  const int64_t pi = ((rq.t0 + i) * a.Hq + h) * a.splits;
  float m = -INFINITY;
  for (int s = tid; s < a.splits; s += D / 2) m = fmaxf(m, a.part_ml[pi + s].x);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  if (D == 128) {
    if (lane == 0) red[0][tid >> 5] = m;
    __syncthreads();
    m = fmaxf(red[0][0], red[0][D / 64 - 1]);
  }
  float sum = 0.0f;
  for (int s = tid; s < a.splits; s += D / 2) {
    const float2 ml = a.part_ml[pi + s];
    // no key: 0, with nothing read; only NaN scores: NaN
    const float w = ml.x == -INFINITY ? ml.y : ex2(ml.x - m);
    f[s] = w;
    sum = fmaf(w, ml.y, sum);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  if (D == 128) {
    if (lane == 0) red[1][tid >> 5] = sum;
    __syncthreads();
    sum = red[1][0] + red[1][D / 64 - 1];
  } else {
    __syncwarp();
  }
  float x = 0.0f, y = 0.0f;
  const float2* src = reinterpret_cast<const float2*>(a.part_o + pi * D) + tid;
#pragma unroll 8
  for (int s = 0; s < a.splits; ++s) {
    const float w = f[s];
    if (w != 0.0f) {
      const float2 v = src[s * (D / 2)];
      x = fmaf(w, v.x, x);
      y = fmaf(w, v.y, y);
    }
  }
  const float inv = m == -INFINITY && sum == 0.0f ? 0.0f : 1.0f / sum;
  *(reinterpret_cast<uint32_t*>(static_cast<uint16_t*>(a.o) + (rq.t0 + i) * a.ldo + static_cast<int64_t>(h) * D) + tid) =
      pack2<BF16>(x * inv, y * inv);
}

template <int D, bool BF16>
cudaError_t launch_join(const PagedArgs& a, cudaStream_t s) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(a.max_q * a.Hq), static_cast<unsigned>(a.B));
  cfg.blockDim = dim3(D / 2);
  cfg.stream = s;
  cudaLaunchAttribute early{};
  early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  early.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &early;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, paged_join_kernel<D, BF16>, a);
}

template <int D, bool BF16, int RT>
cudaError_t launch_rows_t(const PagedArgs& a, cudaStream_t s) {
  using S = RowsShape<D, RT>;
  auto kern = paged_rows_kernel<D, BF16, RT>;
  static bool attr_set[64] = {};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return cudaErrorInvalidDevice;
  if (!attr_set[dev]) {
    const cudaError_t e =
        cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, S::BYTES);
    if (e != cudaSuccess) return e;
    // all of the SM's memory as shared memory: three CTAs of 32 rows need it
    const cudaError_t e2 = cudaFuncSetAttribute(kern, cudaFuncAttributePreferredSharedMemoryCarveout, 100);
    if (e2 != cudaSuccess) return e2;
    attr_set[dev] = true;
  }
  const int64_t tiles = (a.max_q * a.G + 16 * RT - 1) / (16 * RT);
  if (tiles * a.splits > INT32_MAX) return cudaErrorInvalidValue;
  const dim3 grid(static_cast<unsigned>(tiles * a.splits), static_cast<unsigned>(a.Hkv), static_cast<unsigned>(a.B));
  kern<<<grid, kRowsThreads, S::BYTES, s>>>(a, static_cast<int>(tiles));
  const cudaError_t e = cudaGetLastError();
  return e != cudaSuccess || a.splits == 1 ? e : launch_join<D, BF16>(a, s);
}

template <int D, bool BF16>
cudaError_t launch_rows(const PagedArgs& a, cudaStream_t s) {
  return a.max_q * a.G <= 16 ? launch_rows_t<D, BF16, 1>(a, s) : launch_rows_t<D, BF16, 2>(a, s);
}

}  // namespace

// Which kernel, and how the keys are split.  Up to 32 rows a (request, kv head)
// the rows kernel; above, its CTAs would read the keys from the L2 once more for
// every 32 rows, and the tile kernel takes 256 rows at a time.
PagedPlan paged_plan(int64_t B, int64_t T, int64_t max_q, int64_t max_kv, int64_t Hq, int64_t Hkv, int64_t D,
                     bool causal, int64_t window, int64_t sinks) {
  PagedPlan p;
  const int64_t G = Hq / Hkv, rows = max_q * G;
  p.tiles = rows > 32 && G <= kTileRows;
  const int unit = p.tiles ? kTileKeys : kUnit;
  const int64_t tile_rows = p.tiles ? 2 * (kTileRows / G) * G : rows <= 16 ? 16 : 32;
  // Keys that the rows of one CTA can see, in units.
  int64_t span = max_kv;
  if (causal && window > 0 && window + tile_rows + sinks < span) span = window + tile_rows + sinks;
  const int64_t units = span / unit + 3;
  const int64_t ctas = B * Hkv * ((rows + tile_rows - 1) / tile_rows);
  // Rows kernel: the 148 SMs hold two CTAs of 16 rows each, or three of 32.  Requests whose rows all see about
  // as many keys (one request, or a window shorter than they are) are cut into as
  // many stretches as make one wave; others, whose lengths differ, into finer ones,
  // up to eight waves where all are as long as announced (64 requests of 1k to 24k
  // keys: 901 us with one wave, 662 with four, 631 with eight; one of 120k: 111,
  // 142 and 187).  None is shorter than 1024 keys (512 with 32 rows, which are
  // slower work), or joining costs more than it saves.  Tile kernel (one CTA per SM): split only while CTAs are fewer than SMs,
  // into stretches of 512 keys or more.
  const bool alike = B == 1 || span < max_kv;
  const int64_t wave = p.tiles ? 148 : 148 * (rows <= 16 ? 2 : 3);
  const int64_t goal = p.tiles || alike ? wave : wave * (B < 8 ? (B > 0 ? B : 1) : 8);
  const int64_t least = p.tiles ? 512 / kTileKeys : (rows <= 16 ? 1024 : 512) / kUnit;
  int64_t splits = ctas >= goal ? 1 : goal / (ctas > 0 ? ctas : 1);  // (one CTA more than a wave would be two waves)
  if (splits > units / least) splits = units / least;
  if (splits > kJoinMax) splits = kJoinMax;
  if (splits < 1) splits = 1;
  p.split_units = (units + splits - 1) / splits;
  p.splits = (units + p.split_units - 1) / p.split_units;
  if (p.splits > 1) {
    p.part_o_bytes = round_up(T * Hq * p.splits * D * 4, 256);
    p.part_ml_bytes = round_up(T * Hq * p.splits * 8, 256);
  }
  return p;
}

cudaError_t launch_paged_join(const PagedArgs& a, int D, bool bf16, cudaStream_t s) {
  if (D == 64) return bf16 ? launch_join<64, true>(a, s) : launch_join<64, false>(a, s);
  return bf16 ? launch_join<128, true>(a, s) : launch_join<128, false>(a, s);
}

cudaError_t launch_attention_paged(const PagedArgs& a, int D, bool bf16, bool tiles, cudaStream_t s) {
  if (tiles && a.n_pages > 0) return launch_paged_tiles(a, D, bf16, s);
  PagedArgs r = a;
  if (a.n_pages == 0) r.splits = 1;  // no keys at all
  if (D == 64) return bf16 ? launch_rows<64, true>(r, s) : launch_rows<64, false>(r, s);
  return bf16 ? launch_rows<128, true>(r, s) : launch_rows<128, false>(r, s);
}

}  // namespace b2q
