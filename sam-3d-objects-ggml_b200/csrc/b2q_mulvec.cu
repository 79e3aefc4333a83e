// b2q_mulvec.cu -- products of at most kMulVecMaxM tokens with a 4-bit weight
// whose values are taken as they stand (no 8-bit rounding of the activations):
//   Q4_0 (compact layout)  y[m][n] = sum_b d[n,b] sum_i (q_i - 8) x[m][i]
//   Q4_K (GGUF rows)       y[m][n] = sum_s d sc_s sum_i q_i x[m][i] - dmin mn_s sum_i x[m][i]
// then bias, gate and residual as the other few-token product has them.
//
// Bound by the weight's bytes, 0.5625 a value: at the copy rate an SM gets 41
// values a clock, so a value may cost at most three of its 128 lane
// instructions.  Converting codes to floats one by one costs more than that,
// even for one token.  Instead every 32-value block is one int8 matrix product
// (m16n8k32: 16 weight rows, 32 values), which takes the codes as they come out
// of two masks: the nibble layout of both formats is the layout of the A operand.
// The activations become its B operand exactly enough: per token and 32-value
// block a power of two s with |x| / s <= 8355711 (the largest number of three
// balanced base-256 digits), x = s (65536 p0 + 256 p1 + p2) with signed 8-bit
// digits, an absolute error of at most s / 2 <= 2^-23 of the block's largest
// magnitude -- half an ulp of an fp32 number of that size.  The block sums are
// exact in int32; they are read as fp32 through an accumulator that starts at
// the bits of 1.5 * 2^23 (|sum| < 2^22), scaled and added in fp32.
//
// One CTA per SM, 16 warps.  The activations of a run of K ("chunk") are split
// into digits once per CTA and stay in shared memory; then the CTA walks its
// row tiles.  A warp's unit is 16 rows x 256 values, fetched with cp.async into
// the warp's own ring: no barrier inside a tile.  The warps of a tile share out
// its units (WK of them; the other factor of 16, WR, is row tiles side by
// side) and are summed at its end in a fixed order.
//   up to 2 tokens (WIDE false): the 8 columns of one product are token x digit
//   3 to 8 tokens (WIDE true): one product per digit, columns are tokens
#include "b2q_internal.h"
#include "b2q_ptx.cuh"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

namespace b2q {

namespace {

constexpr int kMvWarps = 16, kMvThreads = kMvWarps * 32;
constexpr int kMvStages = 3;
constexpr int kMvUnitK = 256;
constexpr int kMvUnitBytes = 16 * 144;   // Q4_K: 16 rows of a super-block; Q4_0: 2048 of nibbles + 256 of scales
constexpr int kMvTiles = 32;             // row tiles whose sums a CTA keeps while it walks the chunks
constexpr int kMvXBytes = 76 * 1024;     // shared memory for a chunk's activations
constexpr int kMvRing = kMvWarps * kMvStages * kMvUnitBytes;
constexpr int kMvRed = 2 * kMvWarps * 16 * 8 * 4;
constexpr int kMvAcc = kMvTiles * 16 * kMulVecMaxM * 4;
constexpr int kMvMagic = 0x4B400000;     // bits of 1.5 * 2^23

struct MvPlan {
  int wk_shift;        // log2(WK)
  int units;           // of 256 values along K
  int chunk_units;     // of one chunk
  int chunks;
  int64_t supers;      // super-tiles of WR * 16 rows
  int pitch;           // bytes of one digit row in shared memory
  int vec;             // x rows can be read four values at a time
};

template <int XT>
__device__ __forceinline__ float4 x4(const void* x, int64_t i, bool vec) {
  float4 v;
  if constexpr (XT == kXF32) {
    const float* p = static_cast<const float*>(x) + i;
    if (vec) return __ldg(reinterpret_cast<const float4*>(p));
    v = make_float4(__ldg(p), __ldg(p + 1), __ldg(p + 2), __ldg(p + 3));
  } else {
    const uint16_t* p = static_cast<const uint16_t*>(x) + i;
    uint32_t a, b;
    if (vec) {
      const uint2 u = __ldg(reinterpret_cast<const uint2*>(p));
      a = u.x, b = u.y;
    } else {
      a = __ldg(p) | (static_cast<uint32_t>(__ldg(p + 1)) << 16);
      b = __ldg(p + 2) | (static_cast<uint32_t>(__ldg(p + 3)) << 16);
    }
    if constexpr (XT == kXF16) {
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&a));
      const float2 h = __half22float2(*reinterpret_cast<const __half2*>(&b));
      v = make_float4(f.x, f.y, h.x, h.y);
    } else {
      v = make_float4(__uint_as_float(a << 16), __uint_as_float(a & 0xffff0000u), __uint_as_float(b << 16),
                      __uint_as_float(b & 0xffff0000u));
    }
  }
  return v;
}

// 2^e as fp32, -149 <= e <= 127.
__device__ __forceinline__ float pow2(int e) {
  return e >= -126 ? __int_as_float((e + 127) << 23) : __int_as_float(1 << (e + 149));
}

template <bool UNSIGNED_A>
__device__ __forceinline__ void mma_i8_16832(int (&d)[4], const uint32_t (&a)[4], uint2 b) {
  if constexpr (UNSIGNED_A)
    asm volatile(
        "mma.sync.aligned.m16n8k32.row.col.s32.u8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
        : "=r"(d[0]), "=r"(d[1]), "=r"(d[2]), "=r"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b.x), "r"(b.y), "r"(kMvMagic));
  else
    asm volatile(
        "mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
        : "=r"(d[0]), "=r"(d[1]), "=r"(d[2]), "=r"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b.x), "r"(b.y), "r"(kMvMagic));
}

__device__ __forceinline__ void mv_cp16(uint32_t dst, const void* src, bool real) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(real ? 16 : 0) : "memory");
}

template <bool Q4K, bool WIDE, int XT>
__global__ void __launch_bounds__(kMvThreads, 1) mul_vec_kernel(const MulVecArgs a, const MvPlan p) {
  extern __shared__ __align__(128) uint8_t mv_smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, c = lane & 3;
  const int WK = 1 << p.wk_shift, WR = kMvWarps >> p.wk_shift;
  const int wk = warp & (WK - 1), wr = warp >> p.wk_shift;
  const int cols = 3 * a.M;
  uint8_t* ring = mv_smem + warp * kMvStages * kMvUnitBytes;
  const uint32_t ring_a = smem_u32(ring);
  float* red = reinterpret_cast<float*>(mv_smem + kMvRing);          // [2][warp][16][8]
  float* acc_s = reinterpret_cast<float*>(mv_smem + kMvRing + kMvRed);  // [tile][16][M]
  uint8_t* xs = mv_smem + kMvRing + kMvRed + kMvAcc;
  uint8_t* digits = xs;                                              // [col][pitch], digit-major columns when WIDE
  const int nb_chunk = p.chunk_units * (kMvUnitK / 32);
  // per block: WIDE: s of each token; else s times the digit's weight of each column
  float* tab = reinterpret_cast<float*>(xs + static_cast<int64_t>(cols) * p.pitch);
  float* sums = tab + nb_chunk * 8;                    // Q4_K: sum of x per token (WIDE) or column

  const int64_t own = blockIdx.x < p.supers ? (p.supers - blockIdx.x + gridDim.x - 1) / gridDim.x : 0;
  const int group = kMvTiles / WR;  // super-tiles whose sums are kept at once (all, when there is one chunk)
  const int64_t group_n = p.chunks == 1 ? own : group;

  // The warp's sequence of units: for each group, each chunk, each super-tile, its units of the chunk.
  struct Seq {
    int64_t g0, i;
    int chunk, u;
  };
  auto settle = [&](Seq& s) {  // to the next unit that exists, from (g0, i, chunk, u) on
    while (s.g0 < own) {
      const int end = min(p.units, (s.chunk + 1) * p.chunk_units);
      if (s.u < end) return;
      s.u = s.chunk * p.chunk_units + wk;
      if (++s.i >= min(own, s.g0 + group_n)) {
        if (++s.chunk == p.chunks) {
          s.chunk = 0;
          s.g0 += group_n;
        }
        s.i = s.g0;
        s.u = s.chunk * p.chunk_units + wk;
      }
    }
  };
  auto load = [&](const Seq& s, int stage) {
    if (s.g0 < own) {
      const int64_t n0 = ((blockIdx.x + s.i * gridDim.x) * WR + wr) * 16;
      const uint32_t dst = ring_a + stage * kMvUnitBytes;
      if constexpr (Q4K) {
        const uint8_t* src = a.w + n0 * a.row_bytes + static_cast<int64_t>(s.u) * kQ4KBytes;
#pragma unroll
        for (int j = 0; j < 5; ++j) {
          const int x = lane + 32 * j;
          const int r = x / 9, ch = x - 9 * r;
          const bool real = n0 + r < a.N;
          if (x < 144) mv_cp16(dst + x * 16, real ? src + r * a.row_bytes + ch * 16 : a.w, real);
        }
      } else {
        const int64_t k2 = a.K / 2;
        const int ch = lane & 7;
        const bool in_k = s.u * (kMvUnitK / 2) + ch * 16 < k2;
        const uint8_t* src = a.w + static_cast<int64_t>(s.u) * (kMvUnitK / 2) + ch * 16;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int r = (lane >> 3) + 4 * j;
          const bool real = in_k && n0 + r < a.N;
          mv_cp16(dst + r * 128 + ((ch ^ r) & 7) * 16, real ? src + (n0 + r) * k2 : a.w, real);
        }
        if (lane < 16) {
          const int64_t blk = static_cast<int64_t>(s.u) * 8 + (lane >> 1), n8 = n0 + (lane & 1) * 8;
          const bool real = blk < a.K / 32 && n8 < a.lds;
          mv_cp16(dst + 2048 + lane * 16, real ? a.scales + blk * a.lds + n8 : a.scales, real);
        }
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };

  Seq pre{0, 0, 0, wk};
  settle(pre);
#pragma unroll
  for (int s = 0; s < kMvStages - 1; ++s) {
    load(pre, s);
    pre.u += WK;
    settle(pre);
  }
  int stage = 0, fill = kMvStages - 1, buf = 0;

  for (int64_t g0 = 0; g0 < own; g0 += group_n) {
    for (int chunk = 0; chunk < p.chunks; ++chunk) {
      const int cu0 = chunk * p.chunk_units, cu1 = min(p.units, cu0 + p.chunk_units);
      if (p.chunks > 1 || g0 == 0) {
        // ---- the chunk's activations: eight lanes per (token, block), four values each
        const int nb = (cu1 - cu0) * (kMvUnitK / 32);
        for (int j = threadIdx.x >> 3; j < nb * a.M; j += kMvThreads / 8) {
          const int m = j / nb, b = j - m * nb, i = threadIdx.x & 7;
          const int64_t k0 = (static_cast<int64_t>(cu0) * (kMvUnitK / 32) + b) * 32 + i * 4;
          float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
          if (k0 < a.K) v = x4<XT>(a.x, m * a.ldx + k0, p.vec != 0);
          float amax = fmaxf(fmaxf(fabsf(v.x), fabsf(v.y)), fmaxf(fabsf(v.z), fabsf(v.w)));
          // a NaN counts as an infinity (fmaxf would drop it)
          if (!(fabsf(v.x) + fabsf(v.y) + fabsf(v.z) + fabsf(v.w) >= 0.0f)) amax = INFINITY;
          const unsigned mask = 0xffu << (lane & 24);
#pragma unroll
          for (int o = 4; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(mask, amax, o));
          const bool fin = amax < INFINITY;
          int e = static_cast<int>(__float_as_uint(amax) >> 23) - 127 - 22;  // amax in [2^(e+22), 2^(e+23)), or less
          // s = 2^e, and what enters the table (for Q4_0 a sixteenth of it) is an fp32 number
          constexpr int e_min = Q4K ? -149 : -145;
          if (!fin) e = 0;
          if (e >= e_min && amax * pow2(-e / 2) * pow2(-e - -e / 2) > 8355711.0f) ++e;
          if (e < e_min) e = e_min;
          const float i1 = pow2(-e / 2), i2 = pow2(-e - -e / 2);
          int q[4] = {0, 0, 0, 0};
          if (fin) {
            q[0] = __float2int_rn(v.x * i1 * i2);
            q[1] = __float2int_rn(v.y * i1 * i2);
            q[2] = __float2int_rn(v.z * i1 * i2);
            q[3] = __float2int_rn(v.w * i1 * i2);
          }
          uint32_t d0 = 0, d1 = 0, d2 = 0;
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            const int lo = static_cast<int8_t>(q[x]);
            const int hi = (q[x] - lo) >> 8;
            const int mid = static_cast<int8_t>(hi);
            d2 |= (lo & 255u) << (8 * x);
            d1 |= (mid & 255u) << (8 * x);
            d0 |= (((hi - mid) >> 8) & 255u) << (8 * x);
          }
          // lane c of the product reads words (4c ..) and (16 + 4c ..) together
          const int at = b * 32 + (i & 3) * 8 + (i >> 2) * 4;
          const int c0 = WIDE ? m : 3 * m, cs = WIDE ? a.M : 1;
          *reinterpret_cast<uint32_t*>(digits + static_cast<int64_t>(c0) * p.pitch + at) = d0;
          *reinterpret_cast<uint32_t*>(digits + static_cast<int64_t>(c0 + cs) * p.pitch + at) = d1;
          *reinterpret_cast<uint32_t*>(digits + static_cast<int64_t>(c0 + 2 * cs) * p.pitch + at) = d2;
          int xsum = 0;
          if constexpr (Q4K) {  // |sum| <= 32 * 2^23
            xsum = (q[0] + q[1]) + (q[2] + q[3]);
#pragma unroll
            for (int o = 4; o > 0; o >>= 1) xsum += __shfl_xor_sync(mask, xsum, o);
          }
          if (i == 0) {
            // Q4_0 codes go in as 16 (q - 8)
            const float s = fin ? pow2(Q4K ? e : e - 4) : __int_as_float(0x7fc00000);
            if constexpr (WIDE) {
              tab[b * 8 + m] = s;
              if constexpr (Q4K) sums[b * 8 + m] = s * static_cast<float>(xsum);
            } else {
              tab[b * 8 + 3 * m] = s * 65536.0f;
              tab[b * 8 + 3 * m + 1] = s * 256.0f;
              tab[b * 8 + 3 * m + 2] = s;
              if constexpr (Q4K) {
                sums[b * 8 + 3 * m] = s * static_cast<float>(xsum);
                sums[b * 8 + 3 * m + 1] = 0.0f;
                sums[b * 8 + 3 * m + 2] = 0.0f;
              }
            }
          }
        }
        // columns past the tokens: their products are scaled by 0
        const int used = WIDE ? a.M : cols;
        for (int j = threadIdx.x; j < nb * (8 - used); j += kMvThreads) {
          const int b = j / (8 - used), x = used + j - b * (8 - used);
          tab[b * 8 + x] = 0.0f;
          if constexpr (Q4K) sums[b * 8 + x] = 0.0f;
        }
        __syncthreads();
      }

      for (int64_t i = g0; i < min(own, g0 + group_n); ++i) {
        float acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};  // (row g, columns 2c, 2c+1), (row g + 8, ...)
        // B operand: this lane's column is g (of the digit's eight when WIDE)
        const uint8_t* bcol = digits + static_cast<int64_t>(WIDE ? min(g, a.M - 1) : min(g, cols - 1)) * p.pitch + c * 8;
        for (int u = cu0 + wk; u < cu1; u += WK) {
          asm volatile("cp.async.wait_group %0;" ::"n"(kMvStages - 2) : "memory");
          __syncwarp();
          load(pre, fill);
          pre.u += WK;
          settle(pre);
          const uint8_t* st = ring + stage * kMvUnitBytes;
          const int kb0 = (u - cu0) * 8;
          // one block: A operand, scales, table row -> acc
          auto fold = [&](const uint32_t (&af)[4], int kb, float ds0, float ds1, float dm0, float dm1) {
            if constexpr (WIDE) {
              int s0[4], s1[4], s2[4];
              const int64_t ps = static_cast<int64_t>(a.M) * p.pitch;
              mma_i8_16832<Q4K>(s0, af, *reinterpret_cast<const uint2*>(bcol + kb * 32));
              mma_i8_16832<Q4K>(s1, af, *reinterpret_cast<const uint2*>(bcol + ps + kb * 32));
              mma_i8_16832<Q4K>(s2, af, *reinterpret_cast<const uint2*>(bcol + 2 * ps + kb * 32));
              const float2 s = *reinterpret_cast<const float2*>(tab + kb * 8 + 2 * c);
              float2 sx = make_float2(0.0f, 0.0f);
              if constexpr (Q4K) sx = *reinterpret_cast<const float2*>(sums + kb * 8 + 2 * c);
#pragma unroll
              for (int x = 0; x < 4; ++x) {
                const float v = fmaf(__int_as_float(s0[x]) - 12582912.0f, 65536.0f,
                                     fmaf(__int_as_float(s1[x]) - 12582912.0f, 256.0f,
                                          __int_as_float(s2[x]) - 12582912.0f));
                const float d = x < 2 ? ds0 : ds1;
                acc[x] = fmaf(v * ((x & 1) ? s.y : s.x), d, acc[x]);
                if constexpr (Q4K) acc[x] = fmaf(x < 2 ? dm0 : dm1, (x & 1) ? sx.y : sx.x, acc[x]);
              }
            } else {
              int s[4];
              mma_i8_16832<Q4K>(s, af, *reinterpret_cast<const uint2*>(bcol + kb * 32));
              const float2 f = *reinterpret_cast<const float2*>(tab + kb * 8 + 2 * c);
#pragma unroll
              for (int x = 0; x < 4; ++x)
                acc[x] = fmaf((__int_as_float(s[x]) - 12582912.0f) * ((x & 1) ? f.y : f.x), x < 2 ? ds0 : ds1, acc[x]);
              if constexpr (Q4K) {
                const float2 sx = *reinterpret_cast<const float2*>(sums + kb * 8 + 2 * c);
                acc[0] = fmaf(dm0, sx.x, acc[0]);
                acc[1] = fmaf(dm0, sx.y, acc[1]);
                acc[2] = fmaf(dm1, sx.x, acc[2]);
                acc[3] = fmaf(dm1, sx.y, acc[3]);
              }
            }
          };
          if constexpr (Q4K) {
            // headers of rows g and g + 8: (d, dmin), then the 6-bit scales and minima of the eight blocks
            float d[2], dm[2];
            uint32_t sc[2][2], mn[2][2];
#pragma unroll
            for (int r = 0; r < 2; ++r) {
              const uint4 h = *reinterpret_cast<const uint4*>(st + (g + 8 * r) * 144);
              const float2 dd = __half22float2(*reinterpret_cast<const __half2*>(&h.x));
              d[r] = dd.x;
              dm[r] = -dd.y;
              sc[r][0] = h.y & 0x3f3f3f3fu;
              mn[r][0] = h.z & 0x3f3f3f3fu;
              sc[r][1] = (h.w & 0x0f0f0f0fu) | ((h.y >> 2) & 0x30303030u);
              mn[r][1] = ((h.w >> 4) & 0x0f0f0f0fu) | ((h.z >> 2) & 0x30303030u);
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              uint32_t w[2][2];
#pragma unroll
              for (int r = 0; r < 2; ++r)
#pragma unroll
                for (int x = 0; x < 2; ++x)
                  w[r][x] = *reinterpret_cast<const uint32_t*>(st + (g + 8 * r) * 144 + 16 + 32 * j + 16 * x + 4 * c);
#pragma unroll
              for (int x = 0; x < 2; ++x) {  // low nibbles: block 2j; high ones (16 q): block 2j + 1
                const uint32_t mask = x ? 0xf0f0f0f0u : 0x0f0f0f0fu;
                const uint32_t af[4] = {w[0][0] & mask, w[1][0] & mask, w[0][1] & mask, w[1][1] & mask};
                const int bi = 2 * j + x;
                float ds[2], ms[2];
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                  ds[r] = d[r] * static_cast<float>((sc[r][bi >> 2] >> (8 * (bi & 3))) & 255u) * (x ? 0.0625f : 1.0f);
                  ms[r] = dm[r] * static_cast<float>((mn[r][bi >> 2] >> (8 * (bi & 3))) & 255u);
                }
                fold(af, kb0 + bi, ds[0], ds[1], ms[0], ms[1]);
              }
            }
          } else {
            const uint16_t* sc = reinterpret_cast<const uint16_t*>(st + 2048);
#pragma unroll
            for (int bi = 0; bi < 8; ++bi) {
              const uint32_t w0 = *reinterpret_cast<const uint32_t*>(st + g * 128 + ((bi ^ g) & 7) * 16 + c * 4);
              const uint32_t w1 = *reinterpret_cast<const uint32_t*>(st + (g + 8) * 128 + ((bi ^ g) & 7) * 16 + c * 4);
              const uint32_t af[4] = {((w0 << 4) & 0xf0f0f0f0u) ^ 0x80808080u, ((w1 << 4) & 0xf0f0f0f0u) ^ 0x80808080u,
                                      (w0 & 0xf0f0f0f0u) ^ 0x80808080u, (w1 & 0xf0f0f0f0u) ^ 0x80808080u};
              fold(af, kb0 + bi, __half2float(__ushort_as_half(sc[bi * 16 + g])),
                   __half2float(__ushort_as_half(sc[bi * 16 + g + 8])), 0.0f, 0.0f);
            }
          }
          __syncwarp();  // every lane has read the stage before it is refilled
          stage = stage + 1 == kMvStages ? 0 : stage + 1;
          fill = fill + 1 == kMvStages ? 0 : fill + 1;
        }
        float* mine = red + (buf * kMvWarps + warp) * 128;
        *reinterpret_cast<float2*>(mine + g * 8 + 2 * c) = make_float2(acc[0], acc[1]);
        *reinterpret_cast<float2*>(mine + (g + 8) * 8 + 2 * c) = make_float2(acc[2], acc[3]);
        __syncthreads();  // and the other buffer's readers are done before it is written again
        // Warp w sums rows w, w + 16, .. of the super-tile: lanes over (warp of the tile, column).
        for (int r = warp; r < 16 * WR; r += kMvWarps) {
          const float* part = red + (buf * kMvWarps + ((r >> 4) << p.wk_shift)) * 128 + (r & 15) * 8;
          float v = 0.0f;
          for (int x = lane >> 3; x < WK; x += 4) v += part[x * 128 + (lane & 7)];
          v += __shfl_xor_sync(0xffffffffu, v, 8);
          v += __shfl_xor_sync(0xffffffffu, v, 16);
          if constexpr (!WIDE) {
            const int t3 = 3 * min(lane, a.M - 1);
            const float v0 = __shfl_sync(0xffffffffu, v, t3), v1 = __shfl_sync(0xffffffffu, v, t3 + 1),
                        v2 = __shfl_sync(0xffffffffu, v, t3 + 2);
            v = v0 + (v1 + v2);
          }
          const int64_t n = (blockIdx.x + i * gridDim.x) * WR * 16 + r;
          if (lane < a.M && n < a.N) {
            if (p.chunks > 1) {
              float* slot = acc_s + (static_cast<int>(i - g0) * 16 * WR + r) * a.M + lane;
              if (chunk > 0) v += *slot;
              *slot = v;
            }
            if (chunk == p.chunks - 1) {
              if (a.bias) v = __fadd_rn(v, a.bias[n]);
              if (a.resid) v = __fadd_rn(a.resid[lane * a.ldr + n], a.gate ? __fmul_rn(v, a.gate[n]) : v);
              a.y[lane * a.ldy + n] = v;
            }
          }
        }
        buf ^= 1;
      }
    }
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");
}

template <bool Q4K, bool WIDE, int XT>
cudaError_t launch_mv(const MulVecArgs& a, int num_sms, cudaStream_t s) {
  auto kern = mul_vec_kernel<Q4K, WIDE, XT>;
  MvPlan p{};
  p.units = static_cast<int>((a.K + kMvUnitK - 1) / kMvUnitK);
  // Shared memory per value of K: the digits, and per 32 values the table and the sums.
  const int per_k = 3 * a.M + 1 + (Q4K ? 1 : 0);
  const int most = kMvXBytes / (per_k * kMvUnitK) - 1;  // (the digit rows' padding fits one unit)
  p.chunks = (p.units + most - 1) / most;
  p.chunk_units = (p.units + p.chunks - 1) / p.chunks;
  p.chunks = (p.units + p.chunk_units - 1) / p.chunk_units;
  p.pitch = p.chunk_units * kMvUnitK + 32;
  const int64_t tiles = (a.N + 15) / 16;
  // WK, the warps that share a tile's units: all 16 while that gives each two
  // units of a chunk (long runs per warp keep the sums at a tile's end cheap);
  // fewer rows than SMs: as many as there are units.
  int sh = 4;
  while (sh > 0 && (1 << sh) * 2 > p.chunk_units && tiles > static_cast<int64_t>(num_sms) * (kMvWarps >> sh)) --sh;
  while (sh > 0 && (1 << sh) > p.chunk_units) --sh;
  p.wk_shift = sh;
  const int wr = kMvWarps >> sh;
  p.supers = (tiles + wr - 1) / wr;
  const uintptr_t xa = reinterpret_cast<uintptr_t>(a.x);
  p.vec = XT == kXF32 ? (xa % 16 == 0 && a.ldx % 4 == 0) : (xa % 8 == 0 && a.ldx % 4 == 0);
  const int smem = kMvRing + kMvRed + kMvAcc + kMvXBytes;
  static bool attr_set[64] = {};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return cudaErrorInvalidDevice;
  if (!attr_set[dev]) {
    const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return e;
    attr_set[dev] = true;
  }
  const int64_t grid = p.supers < num_sms ? p.supers : num_sms;
  kern<<<static_cast<unsigned>(grid), kMvThreads, smem, s>>>(a, p);
  return cudaGetLastError();
}

}  // namespace

cudaError_t launch_mul_vec(const MulVecArgs& a, bool q4k, int xt, int num_sms, cudaStream_t s) {
  const bool wide = a.M > 2;
#define B2Q_MV(Q, W)                                                                     \
  (xt == kXF32 ? launch_mv<Q, W, kXF32>(a, num_sms, s)                                   \
               : xt == kXF16 ? launch_mv<Q, W, kXF16>(a, num_sms, s) : launch_mv<Q, W, kXBF16>(a, num_sms, s))
  if (q4k) return wide ? B2Q_MV(true, true) : B2Q_MV(true, false);
  return wide ? B2Q_MV(false, true) : B2Q_MV(false, false);
#undef B2Q_MV
}

}  // namespace b2q
