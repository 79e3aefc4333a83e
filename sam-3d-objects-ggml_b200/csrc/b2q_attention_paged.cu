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
// warps takes 16 rows, or 32 (RT 2), and one stretch of the keys.  Every warp takes
// units of 16 keys in turn, with a ring of cp.async stages of its own (no barrier
// inside the loop), its own running maxima, sums and outputs for all the rows, and
// they join at the end.  With 32 rows an operand of keys serves two products, and q
// comes from shared memory: outputs take the registers.  (Two warps with 16 rows each
// and a shared ring instead, a barrier of the two per unit: 104 us against 88 for 24
// rows over 120k keys, 143 against 117 for 64 requests with heads of 64.  Two CTAs of
// 16 rows read the keys twice: 192 us.)  A unit lies inside one
// page (pages are multiples of 16), keys that no row of the CTA sees are not loaded
// but filled with zeros.  Products are m16n8k16; P is fed to the second product as
// two 16-bit numbers, P and what rounding it left: the tensor pipe idles behind the
// loads, and a single rounding of P would cost as much accuracy as the output's own (two
// bf16 numbers hold P to 2^-17 of it, two fp16 ones to 2^-22).
// Before the first products stand three loads that need one another (lengths, page,
// keys), so the pages of a whole ring are asked for at once, ahead of q: with one
// after the other, and 64-bit row numbers, a CTA took 7 us to its first unit, now 4.5.
// Stretches are split over CTAs when the rows alone do not fill the GPU; a
// second kernel, or the cluster that they form, then joins their outputs by their
// maxima and sums.
// Measured (32 / 8 heads of 128): 64 requests of 0.9k to 24k keys 476 us,
// 6850 GB/s; one of 120k keys 81 us, 6040 GB/s; 16 requests, 24 / 4 heads, a window of
// 4096 keys, 1 to 5 tokens 35.0 us, 3850 GB/s; 3 requests of 16 heads of 64
// over at most 900 keys 6.1 us, a launch and one CTA's chain of units.
#include "b2q_internal.h"
#include "b2q_paged.cuh"
#include "b2q_ptx.cuh"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <cmath>

namespace b2q {

namespace {

constexpr int kRowsWarps = 4;
constexpr int kRowsThreads = kRowsWarps * 32;
constexpr int kUnit = 16;  // keys
constexpr int kClusterMax = 8;

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
// Two floats of the cluster's CTA `rank`, at this CTA's address of them.
__device__ __forceinline__ float2 ld_cluster(uint32_t addr, int rank) {
  uint32_t there;
  float2 v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(there) : "r"(addr), "r"(rank));
  asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(there) : "memory");
  return v;
}
template <int D, int RT>
struct RowsShape {
  static constexpr int STAGES = D == 64 ? 4 : 3;
  static constexpr int KV = kUnit * D * 2;               // bytes of one unit's keys (or values)
  static constexpr int RING = STAGES * 2 * KV;           // per warp
  static constexpr int Q = RT == 1 ? 0 : 16 * RT * D * 2;  // q rows, where the registers do not hold them
  static constexpr int BYTES = kRowsWarps * RING + Q;
};

template <int D, bool BF16, int RT>
__global__ void __launch_bounds__(kRowsThreads, 2) paged_rows_kernel(const PagedArgs a, const int tiles) {
  using S = RowsShape<D, RT>;
  constexpr int CH = D / 8;         // 16-byte chunks of a row
  constexpr int RPI = 32 / CH;      // rows that a warp copies at a time
  constexpr int COPIES = kUnit / RPI;
  constexpr int ROWS = 16 * RT;     // of the CTA
  extern __shared__ __align__(128) uint8_t rows_smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int b = blockIdx.z, hk = blockIdx.y;
  // (the stretches of a cluster are neighbours)
  const int split = a.cluster ? blockIdx.x % a.splits : blockIdx.x / tiles;
  const int tile = a.cluster ? blockIdx.x / a.splits : blockIdx.x % tiles;
  const Request rq = request_of(a, b);
  // (max_q * Hq is below 2^31: row numbers fit 32 bits, whose divisions cost far less)
  const uint32_t G = a.G, rows = static_cast<uint32_t>(rq.n) * G, r0 = static_cast<uint32_t>(tile) * ROWS;
  if (r0 >= rows) return;
  const int64_t p_lo = rq.first + r0 / G, p_hi = rq.first + min(rows - 1, r0 + ROWS - 1) / G;
  const Units un = units_of(a, rq.len, p_lo, p_hi, kUnit);
  // the last stretch takes what a longer request than announced has left
  const int u_all = static_cast<int>(un.count());
  const int u0 = static_cast<int>(min(static_cast<int64_t>(split) * a.split_units, static_cast<int64_t>(u_all)));
  const int u1 =
      split == a.splits - 1 ? u_all : static_cast<int>(min(static_cast<int64_t>(u_all), u0 + a.split_units));
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");  // the joining kernel may get ready
  if (split > 0 && u0 >= u_all && !a.cluster) {  // no keys in this stretch
    const uint32_t r = r0 + threadIdx.x;
    if (threadIdx.x < ROWS && r < rows)
      a.part_ml[((rq.t0 + r / G) * a.Hq + static_cast<int64_t>(hk) * G + r % G) * a.splits + split] =
          make_float2(-INFINITY, 0.0f);
    return;
  }
  const int su = static_cast<int>(un.su), gap = static_cast<int>(un.wu - un.su);
  auto unit_at = [&](int i) { return i < su ? i : i + gap; };
  const int32_t* table = a.table + static_cast<int64_t>(b) * a.ldt;
  // The page of unit i of the stretch (-1: none).
  auto page_of = [&](int i) -> int32_t {
    return i < u1 ? __ldg(table + ((unit_at(i) * kUnit) >> a.page_shift)) : -1;
  };
  // The warp's units are u0 + warp, + kRowsWarps, ..; the first pages are asked for before all else.
  int next = u0 + warp;
  int32_t first_pages[S::STAGES];
#pragma unroll
  for (int s = 0; s < S::STAGES; ++s) first_pages[s] = page_of(next + s * kRowsWarps);

  // Keys: rows of the CTA see [win_lo, key_end) and [0, sinks); every one sees
  // [full_lo, full_hi) and the sinks below full_hi.
  const int key_end = static_cast<int>(max(int64_t{0}, a.causal ? min(rq.len, p_hi + 1) : rq.len));
  const int win_lo = static_cast<int>(un.win_lo);
  const int full_hi = static_cast<int>(max(int64_t{0}, a.causal ? min(rq.len, p_lo + 1) : rq.len));
  const int full_lo = a.window > 0 ? static_cast<int>(max(int64_t{0}, p_hi - a.window + 1)) : 0;
  const int sinks = a.window > 0 ? static_cast<int>(a.sinks) : 0;

  // Rows of this thread: g and g + 8 of each 16; each sees [lo, hi) and the sinks below hi.
  const int g = lane >> 2, c = lane & 3;
  int lo[RT][2], hi[RT][2];
  uint32_t qf[RT == 1 ? D / 16 : 1][4];  // RT 1: the q operand; else it is read from shared memory
  const uint16_t* qp = static_cast<const uint16_t*>(a.q);
#pragma unroll
  for (int y = 0; y < RT; ++y)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const uint32_t r = r0 + y * 16 + g + 8 * e;
      const bool real = r < rows;
      const uint32_t i = real ? r / G : 0;
      const int64_t pos = rq.first + i;
      hi[y][e] = real ? static_cast<int>(max(int64_t{0}, a.causal ? min(rq.len, pos + 1) : rq.len)) : 0;
      lo[y][e] = a.window > 0 ? static_cast<int>(max(int64_t{0}, pos - a.window + 1)) : 0;
      if constexpr (RT == 1) {
        const uint16_t* src = qp + (rq.t0 + i) * a.ldq + (static_cast<int64_t>(hk) * G + (real ? r - i * G : 0)) * D;
#pragma unroll
        for (int ks = 0; ks < D / 16; ++ks) {
          qf[ks][e] = real ? *reinterpret_cast<const uint32_t*>(src + ks * 16 + 2 * c) : 0u;
          qf[ks][2 + e] = real ? *reinterpret_cast<const uint32_t*>(src + ks * 16 + 8 + 2 * c) : 0u;
        }
      }
    }

  float m[RT][2], l[RT][2], o[RT][D / 8][4];
#pragma unroll
  for (int y = 0; y < RT; ++y) {
    m[y][0] = m[y][1] = -INFINITY;
    l[y][0] = l[y][1] = 0.0f;
#pragma unroll
    for (int j = 0; j < D / 8; ++j) o[y][j][0] = o[y][j][1] = o[y][j][2] = o[y][j][3] = 0.0f;
  }

  uint8_t* ring = rows_smem + warp * S::RING;
  const uint32_t ring_a = smem_u32(ring);
  const int64_t page_elems = static_cast<int64_t>(a.Hkv) * D << a.page_shift;
  const int64_t lane_elems = (static_cast<int64_t>(hk) * D << a.page_shift) + lane * 8;
  const int page_mask = (1 << a.page_shift) - 1;
  // Chunk ch of row r sits at chunk ch ^ (r % 8) of its 128 bytes.  A lane copies
  // chunk lane % CH of rows lane / CH + RPI x; reads keys (lane & 7) + 8 (lane / 16)
  // of K, (lane & 7) + 8 (lane / 8 % 2) of V.
  const int cr = lane / CH, cc = lane % CH;
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

  uint32_t q_a = 0;
  if constexpr (RT > 1) {  // q rows, chunks placed as the keys' are
    uint8_t* qs = rows_smem + kRowsWarps * S::RING;
#pragma unroll
    for (int x = 0; x < ROWS * CH / kRowsThreads; ++x) {
      const uint32_t row = (threadIdx.x + x * kRowsThreads) / CH, ch = threadIdx.x % CH, r = r0 + row, i = r / G;
      const bool real = r < rows;
      cp16(smem_u32(qs) + row * (D * 2) + ((ch & ~7) | ((ch ^ row) & 7)) * 16,
           real ? qp + (rq.t0 + i) * a.ldq + (static_cast<int64_t>(hk) * G + (r - i * G)) * D + ch * 8 : qp, real);
    }
    cp_commit();
    q_a = smem_u32(qs) + (lane & 15) * (D * 2) + (((lane >> 4) ^ lane) & 7) * 16;
  }
#pragma unroll
  for (int s = 0; s < S::STAGES - 1; ++s, next += kRowsWarps) load(next, s, first_pages[s]);
  int32_t next_page = first_pages[S::STAGES - 1];
  if constexpr (RT > 1) {
    cp_wait<S::STAGES - 1>();
    __syncthreads();
  }
  int stage = 0, fill = S::STAGES - 1;
  for (int i = u0 + warp; i < u1; i += kRowsWarps) {
    cp_wait<S::STAGES - 2>();
    __syncwarp();  // the unit is there
    const uint32_t ka = ring_a + stage * 2 * S::KV, va = ka + S::KV;
    const int k0 = unit_at(i) * kUnit;

    const bool page_in = (present >> stage) & 1u;
    const bool full = page_in && k0 + kUnit <= full_hi && (k0 >= full_lo || k0 + kUnit <= sinks);
    const bool mixed = !full && page_in && p_lo < p_hi;
    float s[2][RT][2][4];  // (RT 1) two accumulation chains per 8 keys
#pragma unroll
    for (int y = 0; y < RT; ++y)
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int x = 0; x < 4; ++x) s[0][y][t][x] = s[1][y][t][x] = 0.0f;
#pragma unroll
    for (int ks = 0; ks < D / 16; ++ks) {
      uint32_t kf[4];
      ldsm4(((ka + k_off) ^ ((ks & 3) * 32)) + (ks >> 2) * 128, kf);
      if constexpr (RT == 1) {
        mma16816<BF16>(s[ks & 1][0][0], qf[ks], kf[0], kf[1]);
        mma16816<BF16>(s[ks & 1][0][1], qf[ks], kf[2], kf[3]);
      } else {
#pragma unroll
        for (int y = 0; y < RT; ++y) {
            uint32_t qq[4];
          ldsm4((q_a ^ ((ks & 3) * 32)) + (ks >> 2) * 128 + y * 16 * (D * 2), qq);
          mma16816<BF16>(s[0][y][0], qq, kf[0], kf[1]);
          mma16816<BF16>(s[0][y][1], qq, kf[2], kf[3]);
        }
      }
    }
    {  // refill the stage before this one (its instructions fill the time that the products take)
      const int32_t pg = next_page;
      next_page = page_of(next + kRowsWarps);
      load(next, fill, pg);
      next += kRowsWarps;
    }
    float mx[RT][2];
    bool grow = false;
#pragma unroll
    for (int y = 0; y < RT; ++y)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            float& v = s[0][y][t][2 * e + x];
            v = (RT == 1 ? v + s[1][y][t][2 * e + x] : v) * a.c2;
          }
        if (!full) {
#pragma unroll
          for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int x = 0; x < 2; ++x) {
              const int j = k0 + t * 8 + 2 * c + x;
              if (!(page_in && j < hi[y][e] && (j >= lo[y][e] || j < sinks))) s[0][y][t][2 * e + x] = -INFINITY;
            }
        }
        float v = fmaxf(fmaxf(s[0][y][0][2 * e], s[0][y][0][2 * e + 1]), fmaxf(s[0][y][1][2 * e], s[0][y][1][2 * e + 1]));
        v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 1));
        v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 2));
        mx[y][e] = v;
        // The maximum in use is raised only when a unit exceeds it by 2^8: P stays
        // below 2^8, which 16-bit floats hold as exactly as values below 1.
        grow |= v > m[y][e] + 8.0f || (m[y][e] == -INFINITY && v != -INFINITY);
      }
    if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
      for (int y = 0; y < RT; ++y)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float nm = fmaxf(m[y][e], mx[y][e]);
          const float al = m[y][e] == -INFINITY ? 0.0f : ex2(m[y][e] - nm);
          m[y][e] = nm;
          l[y][e] *= al;
#pragma unroll
          for (int j = 0; j < D / 8; ++j) {
            o[y][j][2 * e] *= al;
            o[y][j][2 * e + 1] *= al;
          }
        }
    }
    uint32_t ph[RT][4], pl[RT][4];
#pragma unroll
    for (int y = 0; y < RT; ++y)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const float base = m[y][e] == -INFINITY ? 0.0f : m[y][e];
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          float& x = s[0][y][t][2 * e];
          float& z = s[0][y][t][2 * e + 1];
          x = ex2(x - base);
          z = ex2(z - base);
          l[y][e] += x + z;
          const uint32_t h2 = pack2<BF16>(x, z);
          const float2 h = unpack2<BF16>(h2);
          ph[y][2 * t + e] = h2;
          pl[y][2 * t + e] = pack2<BF16>(x - h.x, z - h.y);
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
      for (uint32_t left = bad; left; left &= left - 1) {
        const int r = __ffs(left) - 1, j = k0 + r;
        const int src = (lane & ~3) | ((r & 7) >> 1);
        const uint8_t* vr = vs + r * (D * 2);
#pragma unroll
        for (int ye = 0; ye < 2 * RT; ++ye) {
          const int y = ye >> 1, e = ye & 1;
          const float q0 = __shfl_sync(0xffffffffu, r < 8 ? s[0][y][0][2 * e] : s[0][y][1][2 * e], src);
          const float q1 = __shfl_sync(0xffffffffu, r < 8 ? s[0][y][0][2 * e + 1] : s[0][y][1][2 * e + 1], src);
          const float p = (r & 1) ? q1 : q0;
          if (j < hi[y][e] && (j >= lo[y][e] || j < sinks)) {
#pragma unroll
            for (int d = 0; d < D / 8; ++d) {
              const float2 v =
                  unpack2<BF16>(*reinterpret_cast<const uint32_t*>(vr + ((d & ~7) | ((d ^ r) & 7)) * 16 + c * 4));
              o[y][d][2 * e] = fmaf(p, v.x, o[y][d][2 * e]);
              o[y][d][2 * e + 1] = fmaf(p, v.y, o[y][d][2 * e + 1]);
            }
          }
        }
      }
      if (bad) {
        __syncwarp();  // all have added
        for (uint32_t left = bad; left; left &= left - 1)
          if (lane < CH)
            *reinterpret_cast<uint4*>(vs + (__ffs(left) - 1) * (D * 2) + lane * 16) = make_uint4(0, 0, 0, 0);
        __syncwarp();
      }
    }
#pragma unroll
    for (int j = 0; j < D / 16; ++j) {
      uint32_t vf[4];
      ldsm4_t(((va + v_off) ^ ((j & 3) * 32)) + (j >> 2) * 128, vf);
#pragma unroll
      for (int y = 0; y < RT; ++y) {
        mma16816<BF16>(o[y][2 * j], ph[y], vf[0], vf[1]);
        mma16816<BF16>(o[y][2 * j + 1], ph[y], vf[2], vf[3]);
        mma16816<BF16>(o[y][2 * j], pl[y], vf[0], vf[1]);
        mma16816<BF16>(o[y][2 * j + 1], pl[y], vf[2], vf[3]);
      }
    }
    __syncwarp();  // every lane has read the stage before it is refilled
    stage = stage + 1 == S::STAGES ? 0 : stage + 1;
    fill = fill + 1 == S::STAGES ? 0 : fill + 1;
  }
  cp_wait<0>();
  __syncthreads();

  // Join the four warps: [warp][row] (max, sum), then [warp][row][D], rows 8 banks apart.
  constexpr int OP = D + 8;
  float2* ml = reinterpret_cast<float2*>(rows_smem);
  float* ow = reinterpret_cast<float*>(rows_smem) + kRowsWarps * ROWS * 2;
#pragma unroll
  for (int y = 0; y < RT; ++y)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      float v = l[y][e];
      v += __shfl_xor_sync(0xffffffffu, v, 1);
      v += __shfl_xor_sync(0xffffffffu, v, 2);
      const int row = warp * ROWS + y * 16 + g + 8 * e;
      if (c == 0) ml[row] = make_float2(m[y][e], v);
#pragma unroll
      for (int j = 0; j < D / 8; ++j)
        *reinterpret_cast<float2*>(ow + row * OP + j * 8 + 2 * c) = make_float2(o[y][j][2 * e], o[y][j][2 * e + 1]);
    }
  __syncthreads();
  constexpr int TPR = kRowsThreads / ROWS;  // threads per row
  const int part = threadIdx.x % TPR, row = threadIdx.x / TPR;
  const uint32_t r = r0 + row;
  if (r >= rows && !a.cluster) return;
  float M = -INFINITY;
#pragma unroll
  for (int w = 0; w < kRowsWarps; ++w) M = fmaxf(M, ml[w * ROWS + row].x);
  float f[kRowsWarps], sum = 0.0f;
#pragma unroll
  for (int w = 0; w < kRowsWarps; ++w) {
    const float2 x = ml[w * ROWS + row];
    f[w] = x.x == -INFINITY ? x.y * 0.0f : ex2(x.x - M);  // (no finite score: 0, or NaN where one was NaN)
    sum += f[w] * x.y;
  }
  const bool empty = M == -INFINITY && sum == 0.0f;
  auto joined = [&](int d) {  // values d and d + 1 of the row
    float2 x = make_float2(0.0f, 0.0f);
    if (!empty) {
#pragma unroll
      for (int w = 0; w < kRowsWarps; ++w) {
        const float2 v = *reinterpret_cast<const float2*>(ow + (w * ROWS + row) * OP + d);
        if (f[w] != 0.0f) {  // a warp without keys adds nothing, whatever it holds
          x.x = fmaf(f[w], v.x, x.x);
          x.y = fmaf(f[w], v.y, x.y);
        }
      }
    }
    return x;
  };
  // Values d and d + 1 of row rr, of sum `total`, once their NaN are settled.
  auto settle = [&](float2 x, float total, uint32_t rr, int d) {
    if ((x.x != x.x || x.y != x.y) && total == total) {
      const int64_t pos = rq.first + rr / G;
      const int row_hi = static_cast<int>(max(int64_t{0}, a.causal ? min(rq.len, pos + 1) : rq.len));
      const int row_lo = a.window > 0 ? static_cast<int>(max(int64_t{0}, pos - a.window + 1)) : 0;
      const uint2 seen = nonfinite_seen<1, BF16>(a.v + ((static_cast<int64_t>(hk) * D) << a.page_shift) + d, table, a.n_pages,
                                                 a.page_shift, page_elems, D, row_lo, row_hi, sinks);
      if (x.x != x.x) x.x = settled(seen, 0);
      if (x.y != x.y) x.y = settled(seen, 1);
    }
    return x;
  };
  if (a.cluster) {
    // Each CTA leaves its rows where its first warp's were; then the CTAs share out the
    // values and read them from each other.
    __shared__ float2 done[ROWS];
    if (part == 0) done[row] = make_float2(M, sum);
#pragma unroll
    for (int d = part * 2; d < D; d += TPR * 2) *reinterpret_cast<float2*>(ow + row * OP + d) = joined(d);
    asm volatile("barrier.cluster.arrive.release;\nbarrier.cluster.wait.acquire;" ::: "memory");
    const int pairs = static_cast<int>(min(rows - r0, static_cast<uint32_t>(ROWS))) * (D / 2);
    for (int p = split * kRowsThreads + threadIdx.x; p < pairs; p += a.splits * kRowsThreads) {
      const int prow = p / (D / 2), d = p % (D / 2) * 2;
      const uint32_t at_ml = smem_u32(&done[prow]), at_o = smem_u32(ow + prow * OP + d);
      float2 sm[kClusterMax], so[kClusterMax];
#pragma unroll
      for (int w = 0; w < kClusterMax; ++w) {
        sm[w] = make_float2(-INFINITY, 0.0f);
        so[w] = make_float2(0.0f, 0.0f);
        if (w < a.splits) sm[w] = ld_cluster(at_ml, w), so[w] = ld_cluster(at_o, w);
      }
      float m_all = -INFINITY, l_all = 0.0f;
      float2 x = make_float2(0.0f, 0.0f);
#pragma unroll
      for (int w = 0; w < kClusterMax; ++w) m_all = fmaxf(m_all, sm[w].x);
#pragma unroll
      for (int w = 0; w < kClusterMax; ++w) {
        const float u = sm[w].x == -INFINITY ? sm[w].y * 0.0f : ex2(sm[w].x - m_all);  // (as above)
        l_all = fmaf(u, sm[w].y, l_all);
        if (u != 0.0f) {
          x.x = fmaf(u, so[w].x, x.x);
          x.y = fmaf(u, so[w].y, x.y);
        }
      }
      const float inv = m_all == -INFINITY && l_all == 0.0f ? 0.0f : 1.0f / l_all;
      const uint32_t rr = r0 + prow, i = rr / G;
      x = settle(x, l_all, rr, d);
      *reinterpret_cast<uint32_t*>(static_cast<uint16_t*>(a.o) + (rq.t0 + i) * a.ldo +
                                   (static_cast<int64_t>(hk) * G + (rr - i * G)) * D + d) =
          pack2<BF16>(x.x * inv, x.y * inv);
    }
    // none may go while others read from it
    asm volatile("barrier.cluster.arrive.release;\nbarrier.cluster.wait.acquire;" ::: "memory");
    return;
  }
  const int64_t t = rq.t0 + r / G;
  const int64_t h = static_cast<int64_t>(hk) * G + r % G;
  const bool whole = a.splits == 1;
  const float inv = whole ? (empty ? 0.0f : 1.0f / sum) : 1.0f;
  const int64_t pi = (t * a.Hq + h) * a.splits + split;
  if (!whole && part == 0) a.part_ml[pi] = make_float2(M, sum);
#pragma unroll
  for (int d = part * 2; d < D; d += TPR * 2) {
    const float2 x = settle(joined(d), sum, r, d);
    if (whole)
      *reinterpret_cast<uint32_t*>(static_cast<uint16_t*>(a.o) + t * a.ldo + h * D + d) =
          pack2<BF16>(x.x * inv, x.y * inv);
    else
      *reinterpret_cast<float2*>(a.part_o + pi * D + d) = x;
  }
}

// o = sum_s 2^(m_s - M) O_s / sum_s 2^(m_s - M) l_s over the splits for one
// (token, query head) a CTA: every warp works out M and the sum, adds up its share of the
// splits (one warp a split, a lane's values side by side, loads ahead), and the warps' sums
// are added in their order.  One warp per two values looping over all the splits instead
// took 25 us for 148 splits of 48 rows, as long as the attention itself.
// Launched with the attention kernel still running (it waits before it reads).
constexpr int kJoinMax = 1024;  // splits
constexpr int kJoinWarps = 8;   // of a CTA, at most

template <int D, bool BF16>
__global__ void __launch_bounds__(kJoinWarps * 32) paged_join_kernel(const PagedArgs a) {
  constexpr int V = D / 32;  // values of a lane
  __shared__ __align__(16) float red[kJoinWarps][D];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const Request rq = request_of(a, blockIdx.y);
  const int i = blockIdx.x / a.Hq, h = blockIdx.x - i * a.Hq;
  if (i >= rq.n) return;
  const int64_t pi = ((rq.t0 + i) * a.Hq + h) * a.splits;
  const float2* ml = a.part_ml + pi;
  const float* src = a.part_o + pi * D + lane * V;
  float m = -INFINITY;
  for (int s = lane; s < a.splits; s += 32) m = fmaxf(m, ml[s].x);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  // no key: 0, with nothing read; only NaN scores: NaN
  auto weight = [&](float2 x) { return x.x == -INFINITY ? x.y : ex2(x.x - m); };
  float sum = 0.0f;
  for (int s = lane; s < a.splits; s += 32) sum = fmaf(weight(ml[s]), ml[s].y, sum);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  float acc[V] = {};
#pragma unroll 4
  for (int s = warp; s < a.splits; s += warps) {
    const float w = weight(ml[s]);
    if (w != 0.0f) {
      float v[V];
      if constexpr (V == 4)
        *reinterpret_cast<float4*>(v) = *reinterpret_cast<const float4*>(src + static_cast<int64_t>(s) * D);
      else
        *reinterpret_cast<float2*>(v) = *reinterpret_cast<const float2*>(src + static_cast<int64_t>(s) * D);
#pragma unroll
      for (int x = 0; x < V; ++x) acc[x] = fmaf(w, v[x], acc[x]);
    }
  }
#pragma unroll
  for (int x = 0; x < V; ++x) red[warp][lane * V + x] = acc[x];
  __syncthreads();
  const float inv = m == -INFINITY && sum == 0.0f ? 0.0f : 1.0f / sum;
  uint16_t* to = static_cast<uint16_t*>(a.o) + (rq.t0 + i) * a.ldo + static_cast<int64_t>(h) * D;
  for (int d = 2 * threadIdx.x; d < D; d += 2 * blockDim.x) {
    float x = 0.0f, y = 0.0f;
    for (int w = 0; w < warps; ++w) {
      const float2 v = *reinterpret_cast<const float2*>(&red[w][d]);
      x += v.x;
      y += v.y;
    }
    *reinterpret_cast<uint32_t*>(to + d) = pack2<BF16>(x * inv, y * inv);
  }
}

template <int D, bool BF16>
cudaError_t launch_join(const PagedArgs& a, cudaStream_t s) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(a.max_q * a.Hq), static_cast<unsigned>(a.B));
  cfg.blockDim = dim3(32 * (a.splits >= 4 * kJoinWarps ? kJoinWarps : (a.splits + 3) / 4));
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
    // all of the SM's memory as shared memory: two CTAs of 32 rows need it
    const cudaError_t e2 = cudaFuncSetAttribute(kern, cudaFuncAttributePreferredSharedMemoryCarveout, 100);
    if (e2 != cudaSuccess) return e2;
    attr_set[dev] = true;
  }
  const int64_t tiles = (a.max_q * a.G + 16 * RT - 1) / (16 * RT);
  if (tiles * a.splits > INT32_MAX) return cudaErrorInvalidValue;
  const dim3 grid(static_cast<unsigned>(tiles * a.splits), static_cast<unsigned>(a.Hkv), static_cast<unsigned>(a.B));
  if (a.cluster) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(kRowsThreads);
    cfg.dynamicSmemBytes = S::BYTES;
    cfg.stream = s;
    cudaLaunchAttribute cluster{};
    cluster.id = cudaLaunchAttributeClusterDimension;
    cluster.val.clusterDim.x = static_cast<unsigned>(a.splits);
    cluster.val.clusterDim.y = cluster.val.clusterDim.z = 1;
    cfg.attrs = &cluster;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kern, a, static_cast<int>(tiles));
  }
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
// every 32 rows, and the tile kernel takes 256 rows at a time.  But that one starts
// slower and has one CTA an SM: up to 128 rows over at most 1280 keys stay with the rows
// kernel where one wave holds them (us, rows and tile kernel, 16 heads of 64 and 3
// requests: 40 to 60 rows over 1000 keys 12.5, 24.0; 100 to 120 rows 17.4, 28.1; 40 to 60
// rows over 2900 keys 29.1, 26.1; 3 heads of 128 and 10 requests, 24 to 96 rows over up to
// 2000 keys 25.2, 21.0; 16 requests, 48 to 72 rows in a window of 1000 31.5, 31.0).
PagedPlan paged_plan(int64_t B, int64_t T, int64_t max_q, int64_t max_kv, int64_t Hq, int64_t Hkv, int64_t D,
                     bool causal, int64_t window, int64_t sinks) {
  PagedPlan p;
  const int64_t G = Hq / Hkv, rows = max_q * G;
  const bool brief = rows <= 128 && B * Hkv * ((rows + 31) / 32) <= 148 * 2 &&
                     std::min(max_kv, causal && window > 0 ? window + 32 + sinks : max_kv) <= 1280;
  p.tiles = rows > 32 && G <= kTileRows && !brief;
  const int unit = p.tiles ? kTileKeys : kUnit;
  const int64_t tile_rows = p.tiles ? 2 * (kTileRows / G) * G : rows <= 16 ? 16 : 32;
  // Keys that the rows of one CTA can see, in units.
  int64_t span = max_kv;
  if (causal && window > 0 && window + tile_rows + sinks < span) span = window + tile_rows + sinks;
  const int64_t units = span / unit + 3;
  const int64_t ctas = B * Hkv * ((rows + tile_rows - 1) / tile_rows);
  // Rows kernel: the 148 SMs hold two CTAs each.  Requests whose rows all see about
  // as many keys (one request, or a window shorter than they are) are cut into as
  // many stretches as make one wave; others, whose lengths differ, into finer ones,
  // up to eight waves where all are as long as announced (64 requests of 1k to 24k
  // keys: 901 us with one wave, 662 with four, 631 with eight; one of 120k: 111,
  // 142 and 187).  Past one wave none is shorter than 512 keys, or joining
  // costs more than it saves (16 requests of up to 2000 keys, 8 kv heads: 24.8 us in
  // stretches of 1024, 18.2 of 512; 24 rows each: 30 us of 256, 26 of 512).  Up to one
  // wave 128 keys are enough where there are 512 or more (one request, 8 kv heads of
  // 128, 4k keys: 21.1 us in stretches of 1024, 13.8 of 512, 10.3 of 128, 11.0 of 64;
  // 700 keys: 10.9 whole, 8.3 of 128; 300 keys: 6.8 whole, 8.0 of 128).
  // Up to eight stretches of 64 keys or more that leave an eighth of a wave free (clusters
  // do not fill it to the last CTA) are a cluster that joins in its own memory, from
  // 256 keys on: one launch, which saves a caller 4.5 us of host time and the GPU 2 (300
  // keys: 6.0 us, 700: 6.2 against 8.6 with the joining kernel, 1500: 7.0 and 8.9, 4k: 10.5
  // and 10.6).  Eight stretches are kept although one wave has room for more as long as
  // they have at most 640 keys, 256 with 32 rows (8k keys: 15.8 us and 13.0; 24 rows of 4k
  // keys: 15.2 and 11.3).  Past one wave clusters wait for their slowest CTA (64 requests
  // of up to 24k keys: 576 us against 477).  Tile kernel
  // (one CTA per SM): split only while CTAs are fewer than SMs, into stretches of 512
  // keys or more.
  const bool alike = B == 1 || span < max_kv;
  const int64_t wave = p.tiles ? 148 : 148 * 2;
  const int64_t goal = p.tiles || alike ? wave : wave * (B < 8 ? (B > 0 ? B : 1) : 8);
  const int64_t least = 512 / unit;
  int64_t splits = ctas >= goal ? 1 : goal / (ctas > 0 ? ctas : 1);  // (one CTA more than a wave would be two waves)
  if (splits > units / least) splits = units / least;
  if (!p.tiles && units >= 512 / kUnit && ctas > 0)
    splits = std::max(splits, std::min(wave / ctas, units / (128 / kUnit)));
  if (!p.tiles && ctas > 0 && units >= 256 / kUnit) {
    const int64_t f = std::min({wave * 7 / 8 / ctas, units / (64 / kUnit), int64_t{kClusterMax}});
    if (f >= splits || (f == kClusterMax && units <= f * (rows <= 16 ? 640 : 256) / kUnit))
      splits = f, p.cluster = f > 1;
  }
  if (splits > kJoinMax) splits = kJoinMax;
  if (splits < 1) splits = 1;
  p.split_units = (units + splits - 1) / splits;
  p.splits = (units + p.split_units - 1) / p.split_units;
  if (p.splits <= 1) p.cluster = false;
  if (p.splits > 1 && !p.cluster) {
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
  if (a.n_pages == 0) r.splits = 1, r.cluster = 0;  // no keys at all
  if (D == 64) return bf16 ? launch_rows<64, true>(r, s) : launch_rows<64, false>(r, s);
  return bf16 ? launch_rows<128, true>(r, s) : launch_rows<128, false>(r, s);
}

}  // namespace b2q
