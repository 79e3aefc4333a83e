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
// warps takes 16 or 32 rows and one stretch of the keys; its warps take the
// stretch's units of 16 keys in turn, each with its own ring of cp.async stages
// (no barrier inside the loop), its own running maxima, sums and outputs, and
// they join at the end.  A unit lies inside one page (pages are multiples of
// 16), keys that no row of the CTA sees are not loaded but filled with zeros.
// Products are m16n8k16; P is fed to the second product as two 16-bit numbers,
// P and what rounding it left: the tensor pipe idles behind the loads, and a
// single rounding of P would cost as much accuracy as the output's own.
// Stretches are split over CTAs when the rows alone do not fill the GPU; a
// second kernel then joins their outputs by their maxima and sums.
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
template <int D>
struct RowsShape {
  static constexpr int STAGES = D == 64 ? 4 : 3;
  static constexpr int KV = kUnit * D * 2;               // bytes of one unit's keys (or values)
  static constexpr int RING = STAGES * 2 * KV;           // per warp
  static constexpr int BYTES = kRowsWarps * RING;
};

// MT: 16-row tiles of the CTA.
template <int D, bool BF16, int MT>
__global__ void __launch_bounds__(kRowsThreads) paged_rows_kernel(const PagedArgs a) {
  using S = RowsShape<D>;
  constexpr int CH = D / 8;  // 16-byte chunks of a row
  extern __shared__ __align__(128) uint8_t rows_smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int b = blockIdx.z, hk = blockIdx.y;
  const int tile = blockIdx.x / a.splits, split = blockIdx.x % a.splits;
  const Request rq = request_of(a, b);
  const int64_t rows = rq.n * a.G;
  const int64_t r0 = static_cast<int64_t>(tile) * (16 * MT);
  if (r0 >= rows) return;
  const int64_t i_lo = r0 / a.G, i_hi = min(rows - 1, r0 + 16 * MT - 1) / a.G;
  const int64_t p_lo = rq.first + i_lo, p_hi = rq.first + i_hi;
  const Units un = units_of(a, rq.len, p_lo, p_hi, kUnit);
  const int64_t u_all = un.count();
  // the last stretch takes what a longer request than announced has left
  const int64_t u0 = static_cast<int64_t>(split) * a.split_units;
  const int64_t u1 = split == a.splits - 1 ? u_all : min(u_all, u0 + a.split_units);
  if (split > 0 && u0 >= u_all) return;  // the joining kernel knows

  // Rows of this thread: g and g + 8 of every 16-row tile.
  const int g = lane >> 2, c = lane & 3;
  int64_t pos[MT][2];
  uint32_t qf[MT][D / 16][4];
  const uint16_t* qp = static_cast<const uint16_t*>(a.q);
#pragma unroll
  for (int mt = 0; mt < MT; ++mt)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int64_t r = r0 + mt * 16 + g + 8 * e;
      const bool real = r < rows;
      const int64_t i = real ? r / a.G : 0;
      pos[mt][e] = real ? rq.first + i : kNowhere;
      const uint16_t* src =
          qp + (rq.t0 + i) * a.ldq + (static_cast<int64_t>(hk) * a.G + (real ? r % a.G : 0)) * D;
#pragma unroll
      for (int ks = 0; ks < D / 16; ++ks) {
        qf[mt][ks][e] = real ? *reinterpret_cast<const uint32_t*>(src + ks * 16 + 2 * c) : 0u;
        qf[mt][ks][2 + e] = real ? *reinterpret_cast<const uint32_t*>(src + ks * 16 + 8 + 2 * c) : 0u;
      }
    }

  float m[MT][2], l[MT][2], o[MT][D / 8][4];
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) {
    m[mt][0] = m[mt][1] = -INFINITY;
    l[mt][0] = l[mt][1] = 0.0f;
#pragma unroll
    for (int j = 0; j < D / 8; ++j) o[mt][j][0] = o[mt][j][1] = o[mt][j][2] = o[mt][j][3] = 0.0f;
  }

  uint8_t* ring = rows_smem + warp * S::RING;
  const uint32_t ring_a = smem_u32(ring);
  const int32_t* table = a.table + static_cast<int64_t>(b) * a.ldt;
  const int64_t page_elems = static_cast<int64_t>(a.Hkv) * D << a.page_shift;
  const int64_t head_elems = static_cast<int64_t>(hk) * D << a.page_shift;
  const int64_t key_end = a.causal ? min(rq.len, p_hi + 1) : rq.len;

  // The page of unit index i of this warp's share (-1: none).
  auto page_of = [&](int64_t i) -> int32_t {
    if (i >= u1) return -1;
    return __ldg(table + ((un.at(i) * kUnit) >> a.page_shift));
  };
  auto load = [&](int64_t i, int stage, int32_t page) {
    if (i < u1) {
      const int64_t k0 = un.at(i) * kUnit;
      const bool have = page >= 0 && page < a.n_pages;
      const int64_t off = (have ? static_cast<int64_t>(page) * page_elems : 0) + head_elems +
                          (k0 & ((int64_t{1} << a.page_shift) - 1)) * D;
      const uint32_t kd = ring_a + stage * 2 * S::KV;
#pragma unroll
      for (int x = lane; x < kUnit * CH; x += 32) {
        const int r = x / CH, ch = x % CH;
        const int64_t key = k0 + r;
        const bool real = have && key < key_end && (key >= un.win_lo || key < a.sinks);
        const uint32_t d = kd + r * (D * 2) + ((ch & ~7) | ((ch ^ r) & 7)) * 16;
        cp16(d, a.k + off + x * 8, real);
        cp16(d + S::KV, a.v + off + x * 8, real);
      }
    }
    cp_commit();  // an empty group keeps the count
  };

  // Ring: unit i of this warp is u0 + warp + 4 i.
  int64_t next = u0 + warp;
#pragma unroll
  for (int s = 0; s < S::STAGES - 1; ++s, next += kRowsWarps) load(next, s, page_of(next));
  int32_t next_page = page_of(next);
  int stage = 0, fill = S::STAGES - 1;
  for (int64_t i = u0 + warp; i < u1; i += kRowsWarps) {
    cp_wait<S::STAGES - 2>();
    __syncwarp();
    const int32_t pg = next_page;
    next_page = page_of(next + kRowsWarps);
    load(next, fill, pg);
    next += kRowsWarps;
    const uint32_t ka = ring_a + stage * 2 * S::KV, va = ka + S::KV;
    const int64_t k0 = un.at(i) * kUnit;

    float s[MT][2][4];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
      for (int t = 0; t < 2; ++t) s[mt][t][0] = s[mt][t][1] = s[mt][t][2] = s[mt][t][3] = 0.0f;
    {
      const int row = (lane & 7) + ((lane >> 4) << 3);
#pragma unroll
      for (int ks = 0; ks < D / 16; ++ks) {
        const int ch = ks * 2 + ((lane >> 3) & 1);
        uint32_t kf[4];
        ldsm4(ka + row * (D * 2) + ((ch & ~7) | ((ch ^ row) & 7)) * 16, kf);
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
          mma16816<BF16>(s[mt][0], qf[mt][ks], kf[0], kf[1]);
          mma16816<BF16>(s[mt][1], qf[mt][ks], kf[2], kf[3]);
        }
      }
    }
    // Does every row of the CTA see every key of the unit?
    const int64_t k_last = k0 + kUnit - 1;
    const bool full = k_last < rq.len && (!a.causal || k_last <= p_lo) &&
                      (a.window <= 0 || k0 > p_hi - a.window || k_last < a.sinks);
    const bool page_in = [&] {
      const int32_t p = __ldg(table + (k0 >> a.page_shift));
      return p >= 0 && p < a.n_pages;
    }();
    float mx[MT][2];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            float& v = s[mt][t][2 * e + x];
            v *= a.c2;
            if (!full || !page_in) {
              const int64_t j = k0 + t * 8 + 2 * c + x;
              if (!page_in || !sees(a, pos[mt][e], j, rq.len)) v = -INFINITY;
            }
          }
        float v = fmaxf(fmaxf(s[mt][0][2 * e], s[mt][0][2 * e + 1]), fmaxf(s[mt][1][2 * e], s[mt][1][2 * e + 1]));
        v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 1));
        v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 2));
        mx[mt][e] = v;
      }
    // The maximum in use is raised only when a unit exceeds it by 2^8: P stays
    // below 2^8, which 16-bit floats hold as exactly as values below 1.
    bool grow = false;
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
      for (int e = 0; e < 2; ++e) grow |= mx[mt][e] > m[mt][e] + 8.0f || (m[mt][e] == -INFINITY && mx[mt][e] != -INFINITY);
    if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float nm = fmaxf(m[mt][e], mx[mt][e]);
          const float al = m[mt][e] == -INFINITY ? 0.0f : ex2(m[mt][e] - nm);
          m[mt][e] = nm;
          l[mt][e] *= al;
#pragma unroll
          for (int j = 0; j < D / 8; ++j) {
            o[mt][j][2 * e] *= al;
            o[mt][j][2 * e + 1] *= al;
          }
        }
    }
    uint32_t ph[MT][4], pl[MT][4];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const float base = m[mt][e] == -INFINITY ? 0.0f : m[mt][e];
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          float& x = s[mt][t][2 * e];
          float& y = s[mt][t][2 * e + 1];
          x = ex2(x - base);
          y = ex2(y - base);
          l[mt][e] += x + y;
          const uint32_t hi = pack2<BF16>(x, y);
          const float2 h = unpack2<BF16>(hi);
          ph[mt][2 * t + e] = hi;
          pl[mt][2 * t + e] = pack2<BF16>(x - h.x, y - h.y);
        }
      }
    if (!full && i_lo < i_hi) {
      // Rows of this unit see different keys.  A key that some row does not see
      // may hold an infinity or a NaN, and 0 times that is no 0: such keys leave
      // the tensor product (their values are zeroed in the stage) and are added
      // to the rows that see them one by one.
      uint32_t bad = 0;
#pragma unroll
      for (int x = lane; x < kUnit * CH; x += 32) {
        const uint4 u = *reinterpret_cast<const uint4*>(ring + stage * 2 * S::KV + S::KV + x * 16);
        if (nonfinite2<BF16>(u.x) || nonfinite2<BF16>(u.y) || nonfinite2<BF16>(u.z) || nonfinite2<BF16>(u.w))
          bad |= 1u << (x / CH);
      }
      bad = __reduce_or_sync(0xffffffffu, bad);
      while (bad) {
        const int r = __ffs(bad) - 1;
        bad &= bad - 1;
        const int src = (lane & ~3) | ((r & 7) >> 1);
        uint8_t* vrow = ring + stage * 2 * S::KV + S::KV + r * (D * 2);
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const float p0 = r < 8 ? s[mt][0][2 * e] : s[mt][1][2 * e];
            const float p1 = r < 8 ? s[mt][0][2 * e + 1] : s[mt][1][2 * e + 1];
            const float q0 = __shfl_sync(0xffffffffu, p0, src), q1 = __shfl_sync(0xffffffffu, p1, src);
            const float p = (r & 1) ? q1 : q0;
            if (page_in && sees(a, pos[mt][e], k0 + r, rq.len)) {
#pragma unroll
              for (int j = 0; j < D / 8; ++j) {
                const float2 v =
                    unpack2<BF16>(*reinterpret_cast<const uint32_t*>(vrow + ((j & ~7) | ((j ^ r) & 7)) * 16 + c * 4));
                o[mt][j][2 * e] = fmaf(p, v.x, o[mt][j][2 * e]);
                o[mt][j][2 * e + 1] = fmaf(p, v.y, o[mt][j][2 * e + 1]);
              }
            }
          }
        __syncwarp();
        for (int x = lane; x < CH; x += 32) *reinterpret_cast<uint4*>(vrow + x * 16) = make_uint4(0, 0, 0, 0);
        __syncwarp();
      }
    }
    {
      const int row = (lane & 7) + (((lane >> 3) & 1) << 3);
#pragma unroll
      for (int j = 0; j < D / 16; ++j) {
        const int ch = 2 * j + (lane >> 4);
        uint32_t vf[4];
        ldsm4_t(va + row * (D * 2) + ((ch & ~7) | ((ch ^ row) & 7)) * 16, vf);
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
          mma16816<BF16>(o[mt][2 * j], ph[mt], vf[0], vf[1]);
          mma16816<BF16>(o[mt][2 * j + 1], ph[mt], vf[2], vf[3]);
          mma16816<BF16>(o[mt][2 * j], pl[mt], vf[0], vf[1]);
          mma16816<BF16>(o[mt][2 * j + 1], pl[mt], vf[2], vf[3]);
        }
      }
    }
    __syncwarp();  // every lane has read the stage before it is refilled
    stage = stage + 1 == S::STAGES ? 0 : stage + 1;
    fill = fill + 1 == S::STAGES ? 0 : fill + 1;
  }
  cp_wait<0>();
  __syncthreads();

  // Join the four warps: [warp][row] (max, sum), then [warp][row][D].
  float2* ml = reinterpret_cast<float2*>(rows_smem);
  float* ow = reinterpret_cast<float*>(rows_smem) + kRowsWarps * 16 * 2;
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) {
    if (mt) __syncthreads();
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      float v = l[mt][e];
      v += __shfl_xor_sync(0xffffffffu, v, 1);
      v += __shfl_xor_sync(0xffffffffu, v, 2);
      const int row = g + 8 * e;
      if (c == 0) ml[warp * 16 + row] = make_float2(m[mt][e], v);
#pragma unroll
      for (int j = 0; j < D / 8; ++j)
        *reinterpret_cast<float2*>(ow + (warp * 16 + row) * D + j * 8 + 2 * c) =
            make_float2(o[mt][j][2 * e], o[mt][j][2 * e + 1]);
    }
    __syncthreads();
    constexpr int TPR = kRowsThreads / 16;  // threads per row
    const int row = threadIdx.x / TPR, part = threadIdx.x % TPR;
    const int64_t r = r0 + mt * 16 + row;
    if (r < rows) {
      float M = -INFINITY;
#pragma unroll
      for (int w = 0; w < kRowsWarps; ++w) M = fmaxf(M, ml[w * 16 + row].x);
      float f[kRowsWarps], sum = 0.0f;
#pragma unroll
      for (int w = 0; w < kRowsWarps; ++w) {
        const float2 x = ml[w * 16 + row];
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
          for (int w = 0; w < kRowsWarps; ++w) {
            const float2 v = *reinterpret_cast<const float2*>(ow + (w * 16 + row) * D + d);
            if (f[w] != 0.0f) {  // a warp without keys adds nothing, whatever it holds
              x = fmaf(f[w], v.x, x);
              y = fmaf(f[w], v.y, y);
            }
          }
        }
        if (whole)
          *reinterpret_cast<uint32_t*>(static_cast<uint16_t*>(a.o) + t * a.ldo + h * D + d) =
              pack2<BF16>(x * inv, y * inv);
        else
          *reinterpret_cast<float2*>(a.part_o + pi * D + d) = make_float2(x, y);
      }
    }
  }
}

// One warp per (token, query head): o = sum_s 2^(m_s - M) O_s / sum_s 2^(m_s - M) l_s
// over the splits that hold keys, in their order.
template <int D, bool BF16>
__global__ void __launch_bounds__(128) paged_join_kernel(const PagedArgs a, int tile_rows, int unit) {
  const int lane = threadIdx.x & 31;
  const int b = blockIdx.y;
  const Request rq = request_of(a, b);
  const int64_t idx = static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 5);  // (token, head) of the request
  if (idx >= rq.n * a.Hq) return;
  const int64_t i = idx / a.Hq, h = idx % a.Hq;
  // the split count of the row's tile
  const int64_t r0 = (i * a.G + h % a.G) / tile_rows * tile_rows;
  const int64_t p_lo = rq.first + r0 / a.G, p_hi = rq.first + min(rq.n * a.G - 1, r0 + tile_rows - 1) / a.G;
  const int64_t units = units_of(a, rq.len, p_lo, p_hi, unit).count();
  const int ns = static_cast<int>(
      min(static_cast<int64_t>(a.splits), max(int64_t{1}, (units + a.split_units - 1) / a.split_units)));
  const int64_t pi = ((rq.t0 + i) * a.Hq + h) * a.splits;
  float M = -INFINITY;
  for (int s = lane; s < ns; s += 32) M = fmaxf(M, a.part_ml[pi + s].x);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
  constexpr int E = D / 32;
  float acc[E] = {}, sum = 0.0f;
  {
    for (int s = 0; s < ns; ++s) {
      const float2 ml = a.part_ml[pi + s];
      if (ml.x == -INFINITY && ml.y == 0.0f) continue;  // no key
      const float f = ml.x == -INFINITY ? ml.y : ex2(ml.x - M);  // (only NaN scores: NaN)
      sum = fmaf(f, ml.y, sum);
      const float* src = a.part_o + (pi + s) * D + lane * E;
#pragma unroll
      for (int e = 0; e < E; e += 2) {
        const float2 v = *reinterpret_cast<const float2*>(src + e);
        acc[e] = fmaf(f, v.x, acc[e]);
        acc[e + 1] = fmaf(f, v.y, acc[e + 1]);
      }
    }
  }
  const float inv = M == -INFINITY && sum == 0.0f ? 0.0f : 1.0f / sum;
  uint32_t* dst = reinterpret_cast<uint32_t*>(static_cast<uint16_t*>(a.o) + (rq.t0 + i) * a.ldo + h * D + lane * E);
#pragma unroll
  for (int e = 0; e < E; e += 2) dst[e / 2] = pack2<BF16>(acc[e] * inv, acc[e + 1] * inv);
}

template <int D, bool BF16>
cudaError_t launch_join(const PagedArgs& a, int tile_rows, int unit, cudaStream_t s) {
  const dim3 grid(static_cast<unsigned>((a.max_q * a.Hq + 3) / 4), static_cast<unsigned>(a.B));
  paged_join_kernel<D, BF16><<<grid, 128, 0, s>>>(a, tile_rows, unit);
  return cudaGetLastError();
}

template <int D, bool BF16, int MT>
cudaError_t launch_rows(const PagedArgs& a, cudaStream_t s) {
  auto kern = paged_rows_kernel<D, BF16, MT>;
  static bool attr_set[64] = {};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return cudaErrorInvalidDevice;
  if (!attr_set[dev]) {
    const cudaError_t e =
        cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, RowsShape<D>::BYTES);
    if (e != cudaSuccess) return e;
    attr_set[dev] = true;
  }
  const int64_t tiles = (a.max_q * a.G + 16 * MT - 1) / (16 * MT);
  if (tiles * a.splits > INT32_MAX) return cudaErrorInvalidValue;
  const dim3 grid(static_cast<unsigned>(tiles * a.splits), static_cast<unsigned>(a.Hkv), static_cast<unsigned>(a.B));
  kern<<<grid, kRowsThreads, RowsShape<D>::BYTES, s>>>(a);
  const cudaError_t e = cudaGetLastError();
  return e != cudaSuccess || a.splits == 1 ? e : launch_join<D, BF16>(a, 16 * MT, kUnit, s);
}

template <int D, bool BF16>
cudaError_t launch_paged_t(const PagedArgs& a, cudaStream_t s) {
  // One 16-row tile when the rows fit it: the second tile would only add padding.
  return a.max_q * a.G <= 16 ? launch_rows<D, BF16, 1>(a, s) : launch_rows<D, BF16, 2>(a, s);
}

}  // namespace

// Which kernel, and how the keys are split.  Up to 32 rows a (request, kv head)
// the rows kernel; above, its 32-row tiles would read the keys once more for
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
  // Rows kernel: stretches short enough that the GPU's 148 SMs x 2 CTAs each get
  // eight of them where the requests are alike, and none shorter than 256 keys.
  // Tile kernel (one CTA per SM): split only while CTAs are fewer than SMs, into
  // stretches of 512 keys or more.
  const int64_t goal = p.tiles ? 148 : 148 * 16, least = p.tiles ? 512 / kTileKeys : 16;
  const int64_t want = ctas >= goal ? 1 : p.tiles ? goal / (ctas > 0 ? ctas : 1) : (goal + ctas - 1) / (ctas > 0 ? ctas : 1);
  int64_t per = (units + want - 1) / want;
  if (per < least) per = least;
  if (units <= per) per = units;
  p.split_units = per;
  p.splits = (units + per - 1) / per;
  if (p.splits > 1) {
    p.part_o_bytes = round_up(T * Hq * p.splits * D * 4, 256);
    p.part_ml_bytes = round_up(T * Hq * p.splits * 8, 256);
  }
  return p;
}

cudaError_t launch_paged_join(const PagedArgs& a, int D, bool bf16, int tile_rows, int unit, cudaStream_t s) {
  if (D == 64) return bf16 ? launch_join<64, true>(a, tile_rows, unit, s) : launch_join<64, false>(a, tile_rows, unit, s);
  return bf16 ? launch_join<128, true>(a, tile_rows, unit, s) : launch_join<128, false>(a, tile_rows, unit, s);
}

cudaError_t launch_attention_paged(const PagedArgs& a, int D, bool bf16, bool tiles, cudaStream_t s) {
  if (tiles && a.n_pages > 0) return launch_paged_tiles(a, D, bf16, s);
  PagedArgs r = a;
  if (a.n_pages == 0) r.splits = 1;  // no keys at all
  if (D == 64) return bf16 ? launch_paged_t<64, true>(r, s) : launch_paged_t<64, false>(r, s);
  return bf16 ? launch_paged_t<128, true>(r, s) : launch_paged_t<128, false>(r, s);
}

}  // namespace b2q
