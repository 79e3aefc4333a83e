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
// exact in int32, converted, scaled and added in fp32.
//
// One CTA per SM, 16 or 24 warps.  The activations of a run of K ("chunk") are split
// into digits once per CTA and stay in shared memory; then the CTA walks its
// row tiles.  A warp's unit is 16 rows x 256 values, fetched with cp.async into
// the warp's own ring: no barrier inside a tile.  The warps of a tile share out
// its units (WK of them; the other factor, WR, is row tiles side by
// side) and are summed at its end in a fixed order.  Where rows are long and
// few, the CTAs of a cluster share out K, so that each splits its part of the
// activations only, and add up their sums out of each other's shared memory.
//   up to 4 tokens (NT 1 or 2 products a block, two tokens each): a token's
//     columns are (p0, p1, -, p2), so a lane's pair of sums is 256 p0 + p1, or p2:
//     one number to scale
//   5 to 8 tokens (NT 3, WIDE): one product per digit, columns are tokens; the
//     sums of the highest digit (|sum| < 2^22) are read as fp32 through an
//     accumulator that starts at the bits of 1.5 * 2^23
// Three or four products of the first kind instead, for 5 to 8 tokens, of a
// 49152 x 8192 weight, in steady calls: 157 us against 125 (8 tokens, Q4_K), 111 against 111 (6).
// Measured: that weight in Q4_K, one token: 49 us, 4620 GB/s, 2.5 lane instructions
// a value in 64% of the issue slots; 4 tokens 75 us, 8 tokens 112 us, each token's sums
// to scale and add; 8192 x 4096 Q4_0, 4 tokens: 11.9 us, digits,
// units and a launch in equal parts; 6144 x 1024 Q4_0, one token: 4.5 us, a launch
// and one CTA's chain (the weight's bytes are 0.6 us).
#include "b2q_internal.h"
#include "b2q_ptx.cuh"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>

namespace b2q {

namespace {

constexpr int kMvUnitK = 256;
// A stage: Q4_K 16 super-blocks of 144 bytes; Q4_0 16 rows of 128 bytes of
// nibbles, 16-byte chunks swizzled, and 8 x 16 fp16 scales.  A lane's rows of a
// tile are neighbours: the 8-byte reads of rows 0, 2, 4, 6 (288 bytes apart)
// then meet all banks, and two rows' Q4_0 scales are one word.
constexpr int kMvUnitBytes = 16 * kQ4KBytes;
constexpr int kMvSmem = 227 * 1024;
// The sums of 5 to 8 tokens take more registers a warp, so 16 warps and one more stage each.
template <int NT>
struct MvShape {
  static constexpr bool WIDE = NT == 3;
  static constexpr int TOKENS = WIDE ? 8 : 2 * NT;           // at most
  static constexpr int COLS = WIDE ? 8 : 4 * NT;             // of sums in a lane quad
  static constexpr int WARPS = WIDE ? 16 : 24, THREADS = WARPS * 32;
  static constexpr int STAGES = WIDE ? 3 : 2;
  static constexpr int TILES = 32;                           // row tiles whose sums a CTA keeps over the chunks
  static constexpr int RING = WARPS * STAGES * kMvUnitBytes;
  static constexpr int SCALES = WARPS * 8 * 16 * 4;          // Q4_K: a unit's d * sc per warp
  static constexpr int RED = 2 * WARPS * 16 * COLS * 4;
  static constexpr int ACC = TILES * 16 * TOKENS * 4;
  static constexpr int X = kMvSmem - RING - SCALES - RED - ACC;  // a chunk's activations
};
constexpr int kMvRanks = 8;              // CTAs of a cluster, at most
constexpr int kMvBatch = 4;              // blocks of activations that a group of lanes loads at a time
constexpr int kMvMagic = 0x4B400000;     // bits of 1.5 * 2^23

struct MvPlan {
  int wk, wr;          // warps that share a tile's units, and tiles side by side: WK * WR warps work
  int wk_inv;          // 2^16 / WK rounded up
  int units;           // of 256 values along K
  int chunk_units;     // of one chunk
  int chunks;
  int supers;          // super-tiles of WR * 16 rows; at least one per cluster
  int rank_shift;      // log2 of the CTAs of a cluster
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

// All four sums start at `init`.
template <bool UNSIGNED_A>
__device__ __forceinline__ void mma_i8_16832(int (&d)[4], const uint32_t (&a)[4], uint2 b, int init) {
  if constexpr (UNSIGNED_A)
    asm volatile(
        "mma.sync.aligned.m16n8k32.row.col.s32.u8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
        : "=r"(d[0]), "=r"(d[1]), "=r"(d[2]), "=r"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b.x), "r"(b.y), "r"(init));
  else
    asm volatile(
        "mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
        : "=r"(d[0]), "=r"(d[1]), "=r"(d[2]), "=r"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b.x), "r"(b.y), "r"(init));
}

__device__ __forceinline__ void mv_cp16(uint32_t dst, const void* src, bool real) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(real ? 16 : 0) : "memory");
}

// A float of the cluster's CTA `rank`, at this CTA's address of it.
__device__ __forceinline__ float mv_peer(uint32_t addr, int rank) {
  uint32_t there;
  float v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(there) : "r"(addr), "r"(rank));
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(there) : "memory");
  return v;
}

// CLUSTER: the CTAs of a cluster share out K and add up their sums.
template <bool Q4K, int NT, int XT, bool CLUSTER>
__global__ void __launch_bounds__(MvShape<NT>::THREADS, 1) mul_vec_kernel(const MulVecArgs a, const MvPlan p) {
  using S = MvShape<NT>;
  constexpr bool WIDE = S::WIDE;
  extern __shared__ __align__(128) uint8_t mv_smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, c = lane & 3;
  const int WK = p.wk, WR = p.wr;
  const int wr = warp * p.wk_inv >> 16, wk = warp - wr * WK;  // warp / WK
  const int row0 = 2 * g, row1 = 2 * g + 1;  // of a tile
  uint8_t* ring = mv_smem + warp * S::STAGES * kMvUnitBytes;
  const uint32_t ring_a = smem_u32(ring);
  float* scales = reinterpret_cast<float*>(mv_smem + S::RING) + warp * 128;  // [block % 4][block / 4][row]
  float* red = reinterpret_cast<float*>(mv_smem + S::RING + S::SCALES);        // [2][warp][16][COLS]
  float* acc_s = reinterpret_cast<float*>(mv_smem + S::RING + S::SCALES + S::RED);  // [tile][16][M]
  uint8_t* digits = mv_smem + S::RING + S::SCALES + S::RED + S::ACC;  // [digit][token] (WIDE), [token][digit]; pitch
  // per token, the chunk's blocks: s; then (Q4_K) the sum of the block's x
  const int nb_pitch = p.chunk_units * (kMvUnitK / 32) + 4;  // floats; tokens meet different banks
  float* tab = reinterpret_cast<float*>(digits + 3 * a.M * p.pitch);
  float* sums = tab + a.M * nb_pitch;
  constexpr int TC = S::COLS;

  const int rs = CLUSTER ? p.rank_shift : 0, ranks = 1 << rs;
  const int rank = static_cast<int>(blockIdx.x) & (ranks - 1), cid = static_cast<int>(blockIdx.x) >> rs;
  const int clusters = static_cast<int>(gridDim.x) >> rs;
  const int u_lo = rank * p.units >> rs, u_hi = (rank + 1) * p.units >> rs;  // this CTA's units

  const int own = (p.supers - cid + clusters - 1) / clusters;
  const int group_n = p.chunks == 1 && !CLUSTER ? own : S::TILES / WR;  // super-tiles whose sums are kept at once
  const int outs = 16 * WR * a.M;                                           // of a super-tile

  const int mine_n = wr < WR ? own : 0;  // super-tiles that this warp works on

  // The warp's sequence of units: for each group, each chunk, each super-tile, its units of the chunk.
  int q_g0 = 0, q_i = 0, q_chunk = 0, q_u = u_lo + wk, q_end = min(u_hi, u_lo + p.chunk_units);
  const uint8_t* q_src = nullptr;  // the warp's tile
  int64_t q_n0 = 0;
  uint32_t src_off[5];             // this lane's 16-byte pieces of a unit
  auto enter_tile = [&] {
    q_n0 = ((cid + static_cast<int64_t>(q_i) * clusters) * WR + wr) * 16;
    q_n0 = min(q_n0, (a.N - 1) / 16 * 16);  // (a tile past the end repeats the last one, unused)
    q_src = a.w + q_n0 * a.row_bytes;
    const int last = static_cast<int>(min(a.N - 1 - q_n0, int64_t{15}));
#pragma unroll
    for (int j = 0; j < 5; ++j) {
      const int x = lane + 32 * j;
      if constexpr (Q4K)
        src_off[j] = static_cast<uint32_t>(min(x / 9, last)) * static_cast<uint32_t>(a.row_bytes) + (x % 9) * 16;
      else
        src_off[j] = static_cast<uint32_t>(min(x / 8, last)) * static_cast<uint32_t>(a.row_bytes) + (x % 8) * 16;
    }
  };
  auto settle = [&] {  // to the next unit that exists
    while (q_u >= q_end && q_g0 < mine_n) {
      if (++q_i >= min(own, q_g0 + group_n)) {
        if (++q_chunk == p.chunks) {
          q_chunk = 0;
          q_g0 += group_n;
        }
        q_i = q_g0;
        q_end = min(u_hi, u_lo + (q_chunk + 1) * p.chunk_units);
      }
      q_u = u_lo + q_chunk * p.chunk_units + wk;
      enter_tile();
    }
  };
  auto load = [&](int stage) {
    if (q_g0 < mine_n) {
      const uint32_t dst = ring_a + stage * kMvUnitBytes;
      if constexpr (Q4K) {
        const uint8_t* src = q_src + static_cast<int64_t>(q_u) * kQ4KBytes;
#pragma unroll
        for (int j = 0; j < 4; ++j) mv_cp16(dst + (lane + 32 * j) * 16, src + src_off[j], true);
        if (lane < 16) mv_cp16(dst + (lane + 128) * 16, src + src_off[4], true);
      } else {
        const int ch = lane & 7;
        const bool in_k = q_u * (kMvUnitK / 2) + ch * 16 < a.row_bytes;
        const uint8_t* src = q_src + q_u * (kMvUnitK / 2);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int r = (lane >> 3) + 4 * j;
          mv_cp16(dst + r * 128 + ((ch ^ (r >> 1)) & 7) * 16, in_k ? src + src_off[j] : a.w, in_k);
        }
        if (lane < 16) {
          const int64_t blk = static_cast<int64_t>(q_u) * 8 + (lane >> 1), n8 = q_n0 + (lane & 1) * 8;
          const bool real = blk < a.K / 32 && n8 < a.lds;
          mv_cp16(dst + 2048 + lane * 16, real ? a.scales + blk * a.lds + n8 : a.scales, real);
        }
      }
      q_u += WK;
      settle();
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };

  enter_tile();
  settle();
  // The ring's first loads, behind the first activations' (which would wait for them to pass).
  bool primed = false;
  auto prime = [&] {
    if (primed) return;
    primed = true;
#pragma unroll
    for (int s = 0; s < S::STAGES - 1; ++s) load(s);
  };
  int stage = 0, fill = S::STAGES - 1, buf = 0;

  for (int g0 = 0; g0 < own; g0 += group_n) {
    for (int chunk = 0; chunk < p.chunks; ++chunk) {
      const int cu0 = u_lo + chunk * p.chunk_units, cu1 = min(u_hi, cu0 + p.chunk_units);
      if (p.chunks > 1 || g0 == 0) {
        // ---- the chunk's activations: eight lanes per (token, block), four values each
        const int nb = (cu1 - cu0) * (kMvUnitK / 32);
        constexpr int GROUPS = S::THREADS / 8;
        const int gi = threadIdx.x >> 3, i = threadIdx.x & 7;
        const unsigned mask = 0xffu << (lane & 24);
        // (token, block) after (token, block), blocks of a token in a row, GROUPS apart
        int t_m = gi / nb, t_b = gi - t_m * nb;
        const int d_m = GROUPS / nb, d_b = GROUPS - d_m * nb;
        while (t_m < a.M) {
         float4 vb[kMvBatch];
         int vm[kMvBatch], vk[kMvBatch];
#pragma unroll
         for (int y = 0; y < kMvBatch; ++y) {  // loads under way together
          vm[y] = t_m;
          vk[y] = t_b;
          const int64_t k0 = (static_cast<int64_t>(cu0) * (kMvUnitK / 32) + t_b) * 32 + i * 4;
          vb[y] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
          if (t_m < a.M && k0 < a.K) vb[y] = x4<XT>(a.x, t_m * a.ldx + k0, p.vec != 0);
          t_m += d_m;
          t_b += d_b;
          if (t_b >= nb) t_b -= nb, ++t_m;
         }
         prime();
#pragma unroll
         for (int y = 0; y < kMvBatch; ++y) {
          if (vm[y] >= a.M) break;
          const int m = vm[y], b = vk[y];
          const float4 v = vb[y];
          // Magnitudes compare as their bits do, a NaN above infinity.
          uint32_t amax = max(max(__float_as_uint(v.x) & 0x7fffffffu, __float_as_uint(v.y) & 0x7fffffffu),
                              max(__float_as_uint(v.z) & 0x7fffffffu, __float_as_uint(v.w) & 0x7fffffffu));
#pragma unroll
          for (int o = 4; o > 0; o >>= 1) amax = max(amax, __shfl_xor_sync(mask, amax, o));
          const bool fin = amax < 0x7f800000u;
          // s = 2^e with the largest magnitude in [2^22, 8355711] of it: a mantissa past that
          // number's takes the next power.  What enters the table (for Q4_0 a sixteenth of s)
          // has to be an fp32 number, so e has a lowest value.
          constexpr int e_min = Q4K ? -149 : -145;
          const int e = max(static_cast<int>(amax >> 23) - 149 + ((amax & 0x7fffffu) > 0x7efefeu ? 1 : 0), e_min);
          // 1 / s in two steps, for the sake of e below -126
          const float i1 = __uint_as_float(static_cast<uint32_t>(127 - max(e, -126)) << 23);
          const float i2 = __uint_as_float(static_cast<uint32_t>(127 + max(-126 - e, 0)) << 23);
          int q[4] = {0, 0, 0, 0};
          if (fin) {
            q[0] = __float2int_rn(v.x * i1 * i2);
            q[1] = __float2int_rn(v.y * i1 * i2);
            q[2] = __float2int_rn(v.z * i1 * i2);
            q[3] = __float2int_rn(v.w * i1 * i2);
          }
          // Balanced digits: with 128 (65536 + 256 + 1) added every digit is 128 + p, and
          // flipping its top bit makes the byte p; then bytes of four values into words.
          uint32_t u[4];
#pragma unroll
          for (int x = 0; x < 4; ++x) u[x] = (static_cast<uint32_t>(q[x]) + 0x808080u) ^ 0x808080u;
          const uint32_t a01 = __byte_perm(u[0], u[1], 0x5140), a23 = __byte_perm(u[2], u[3], 0x5140);
          const uint32_t d2 = __byte_perm(a01, a23, 0x5410), d1 = __byte_perm(a01, a23, 0x7632);
          const uint32_t d0 = __byte_perm(__byte_perm(u[0], u[1], 0x0062), __byte_perm(u[2], u[3], 0x0062), 0x5410);
          // Lane c of the product has values 4c .. and 16 + 4c .. (Q4_0) or 8c .. 8c + 7 (Q4_K) of
          // a block; its pieces of two neighbouring blocks are one 16-byte word.
          const int lc = Q4K ? i >> 1 : i & 3, half = Q4K ? i & 1 : i >> 2;
          const int at = (b >> 1) * 64 + lc * 16 + (b & 1) * 8 + half * 4;
          const int c0 = WIDE ? m : 3 * m, cs = WIDE ? a.M : 1;
          *reinterpret_cast<uint32_t*>(digits + c0 * p.pitch + at) = d0;
          *reinterpret_cast<uint32_t*>(digits + (c0 + cs) * p.pitch + at) = d1;
          *reinterpret_cast<uint32_t*>(digits + (c0 + 2 * cs) * p.pitch + at) = d2;
          int xsum = 0;
          if constexpr (Q4K) {  // |sum| <= 32 * 2^23
            xsum = (q[0] + q[1]) + (q[2] + q[3]);
#pragma unroll
            for (int o = 4; o > 0; o >>= 1) xsum += __shfl_xor_sync(mask, xsum, o);
          }
          if (i == 0) {
            // Q4_0 codes go in as 16 (q - 8)
            const float s = fin ? pow2(Q4K ? e : e - 4) : __int_as_float(0x7fc00000);
            tab[m * nb_pitch + b] = s;
            if constexpr (Q4K) sums[m * nb_pitch + b] = s * static_cast<float>(xsum);
          }
         }
        }
        prime();
        __syncthreads();
      }

      // B operand: this lane's column is g; narrow: of products 0 .. NT - 1, digits (p0, p1, p0 unused, p2).
      // Columns past the tokens repeat the last one, unused.
      constexpr int NB = WIDE ? 1 : NT;
      const uint8_t* bcol[NB];
      const float* tab0[NB];                    // s of this lane's token (WIDE: tokens 2c and 2c + 1)
#pragma unroll
      for (int x = 0; x < NB; ++x) {
        const int digit = (g & 3) == 3 ? 2 : (g & 1);
        bcol[x] = digits + (WIDE ? min(g, a.M - 1) : 3 * min(2 * x + (g >> 2), a.M - 1) + digit) * p.pitch + c * 16;
        tab0[x] = tab + min(WIDE ? 2 * c : 2 * x + (c >> 1), a.M - 1) * nb_pitch;
      }
      const float* tab1 = tab + min(2 * c + 1, a.M - 1) * nb_pitch;
      const int dstep = a.M * p.pitch;          // WIDE: to the next digit
      const int mul = (c & 1) ? 0 : 256;        // narrow: weight of the first of the lane's two columns
      for (int i = g0; i < min(own, g0 + group_n); ++i) {
        // A thread finishes outputs (row, token) threadIdx.x, + THREADS, .. of the super-tile, rows in a row;
        // what the first one is added to is on its way while the units run.
        const int64_t n_super = (cid + static_cast<int64_t>(i) * clusters) * WR * 16;
        const int m_first = static_cast<int>(threadIdx.x) / (16 * WR);
        const int64_t n_first = n_super + (static_cast<int>(threadIdx.x) - m_first * 16 * WR);
        float bias_first = 0.0f, gate_first = 1.0f, resid_first = 0.0f;
        if (static_cast<int>(threadIdx.x) < outs && n_first < a.N && chunk == p.chunks - 1 && !CLUSTER) {
          if (a.bias) bias_first = __ldg(a.bias + n_first);
          if (a.gate) gate_first = __ldg(a.gate + n_first);
          if (a.resid) resid_first = a.resid[m_first * a.ldr + n_first];
        }
        float macc[Q4K ? S::TOKENS : 1] = {};  // Q4_K: minima, of row lane % 16, half of the blocks
        float acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};  // WIDE: (row0, tokens 2c, 2c + 1), (row1, ..); else (row0, row1) per product
        for (int u = wr < WR ? cu0 + wk : cu1; u < cu1; u += WK) {
          asm volatile("cp.async.wait_group %0;" ::"n"(S::STAGES - 2) : "memory");
          __syncwarp();
          load(fill);
          const uint8_t* st = ring + stage * kMvUnitBytes;
          const int bu = (u - cu0) * kMvUnitK;
          const int kb0 = (u - cu0) * 8;
          // two blocks: A operands, scales of (row0, row1), s of the token(s) -> acc
          auto fold = [&](const uint32_t (&af)[2][4], int pair, const float2 (&sr)[2], const float (&t0)[NB][2],
                          const float (&t1)[2]) {
            if constexpr (WIDE) {
              const uint4 b0 = *reinterpret_cast<const uint4*>(bcol[0] + bu + pair * 64);
              const uint4 b1 = *reinterpret_cast<const uint4*>(bcol[0] + dstep + bu + pair * 64);
              const uint4 b2 = *reinterpret_cast<const uint4*>(bcol[0] + 2 * dstep + bu + pair * 64);
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                int x0[4], x1[4], x2[4];
                mma_i8_16832<Q4K>(x0, af[h], h ? make_uint2(b0.z, b0.w) : make_uint2(b0.x, b0.y), kMvMagic);
                mma_i8_16832<Q4K>(x1, af[h], h ? make_uint2(b1.z, b1.w) : make_uint2(b1.x, b1.y), 0);
                mma_i8_16832<Q4K>(x2, af[h], h ? make_uint2(b2.z, b2.w) : make_uint2(b2.x, b2.y), 0);
#pragma unroll
                for (int x = 0; x < 4; ++x) {
                  const float v = fmaf(__int_as_float(x0[x]) - 12582912.0f, 65536.0f,
                                       static_cast<float>(x1[x] * 256 + x2[x]));
                  acc[x] = fmaf(v * ((x & 1) ? t1[h] : t0[0][h]), x < 2 ? sr[h].x : sr[h].y, acc[x]);
                }
              }
            } else {
#pragma unroll
              for (int n = 0; n < NB; ++n) {
                const uint4 b0 = *reinterpret_cast<const uint4*>(bcol[n] + bu + pair * 64);
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                  int x[4];
                  mma_i8_16832<Q4K>(x, af[h], h ? make_uint2(b0.z, b0.w) : make_uint2(b0.x, b0.y), 0);
                  acc[2 * n] = fmaf(static_cast<float>(x[0] * mul + x[1]) * t0[n][h], sr[h].x, acc[2 * n]);
                  acc[2 * n + 1] = fmaf(static_cast<float>(x[2] * mul + x[3]) * t0[n][h], sr[h].y, acc[2 * n + 1]);
                }
              }
            }
          };
          if constexpr (Q4K) {  // the unit's scales and minima: lane -> row lane % 16, four blocks
            const int half = lane >> 4, row = lane & 15;
            const uint4 h = *reinterpret_cast<const uint4*>(st + row * kQ4KBytes);
            const float2 dd = __half22float2(*reinterpret_cast<const __half2*>(&h.x));
            const uint32_t sc = half ? (h.w & 0x0f0f0f0fu) | ((h.y >> 2) & 0x30303030u) : h.y & 0x3f3f3f3fu;
            const uint32_t mn = half ? ((h.w >> 4) & 0x0f0f0f0fu) | ((h.z >> 2) & 0x30303030u) : h.z & 0x3f3f3f3fu;
            const float d1 = dd.x * 0.0625f;  // odd blocks' codes are read as 16 q
#pragma unroll
            for (int j = 0; j < 4; ++j)
              scales[j * 32 + lane] = ((j & 1) ? d1 : dd.x) * static_cast<float>((sc >> (8 * j)) & 255u);
            const float m0 = static_cast<float>(mn & 255u), m1 = static_cast<float>((mn >> 8) & 255u),
                        m2 = static_cast<float>((mn >> 16) & 255u), m3 = static_cast<float>(mn >> 24);
#pragma unroll
            for (int m = 0; m < S::TOKENS; ++m) {
              if (m >= a.M) break;
              const float4 sx = *reinterpret_cast<const float4*>(sums + m * nb_pitch + kb0 + half * 4);
              macc[m] = fmaf(-dd.y, fmaf(m0, sx.x, fmaf(m1, sx.y, fmaf(m2, sx.z, m3 * sx.w))), macc[m]);
            }
            __syncwarp();
          }
#pragma unroll
          for (int q = 0; q < 2; ++q) {  // four blocks
            float4 ta[NB], tb;
#pragma unroll
            for (int n = 0; n < NB; ++n) ta[n] = *reinterpret_cast<const float4*>(tab0[n] + kb0 + 4 * q);
            tb = ta[0];
            if constexpr (WIDE) tb = *reinterpret_cast<const float4*>(tab1 + kb0 + 4 * q);
#pragma unroll
            for (int r = 0; r < 2; ++r) {
              const int j = 2 * q + r;  // blocks 2j, 2j + 1
              uint32_t af[2][4];
              float2 sr[2];
              if constexpr (Q4K) {  // low nibbles: block 2j; high ones (16 q): block 2j + 1
                const uint2 w0 = *reinterpret_cast<const uint2*>(st + row0 * kQ4KBytes + 16 + 32 * j + 8 * c);
                const uint2 w1 = *reinterpret_cast<const uint2*>(st + row1 * kQ4KBytes + 16 + 32 * j + 8 * c);
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                  const uint32_t mask = h ? 0xf0f0f0f0u : 0x0f0f0f0fu;
                  af[h][0] = w0.x & mask;
                  af[h][1] = w1.x & mask;
                  af[h][2] = w0.y & mask;
                  af[h][3] = w1.y & mask;
                  sr[h] = *reinterpret_cast<const float2*>(scales + ((2 * j + h) & 3) * 32 + q * 16 + row0);
                }
              } else {
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                  const int bi = 2 * j + h, at = ((bi ^ g) & 7) * 16 + c * 4;
                  const uint32_t w0 = *reinterpret_cast<const uint32_t*>(st + row0 * 128 + at);
                  const uint32_t w1 = *reinterpret_cast<const uint32_t*>(st + row1 * 128 + at);
                  af[h][0] = ((w0 << 4) & 0xf0f0f0f0u) ^ 0x80808080u;
                  af[h][1] = ((w1 << 4) & 0xf0f0f0f0u) ^ 0x80808080u;
                  af[h][2] = (w0 & 0xf0f0f0f0u) ^ 0x80808080u;
                  af[h][3] = (w1 & 0xf0f0f0f0u) ^ 0x80808080u;
                  sr[h] = __half22float2(reinterpret_cast<const __half2*>(st + 2048)[bi * 8 + g]);
                }
              }
              float t0[NB][2];
#pragma unroll
              for (int n = 0; n < NB; ++n) t0[n][0] = r ? ta[n].z : ta[n].x, t0[n][1] = r ? ta[n].w : ta[n].y;
              const float t1[2] = {r ? tb.z : tb.x, r ? tb.w : tb.y};
              fold(af, j, sr, t0, t1);
            }
          }
          __syncwarp();  // every lane has read the stage before it is refilled
          stage = stage + 1 == S::STAGES ? 0 : stage + 1;
          fill = fill + 1 == S::STAGES ? 0 : fill + 1;
        }
        float* mine = red + (buf * S::WARPS + warp) * 16 * TC;
        if constexpr (WIDE) {
          *reinterpret_cast<float2*>(mine + row0 * TC + 2 * c) = make_float2(acc[0], acc[1]);
          *reinterpret_cast<float2*>(mine + row1 * TC + 2 * c) = make_float2(acc[2], acc[3]);
        } else {
          const float f = (c & 1) ? 1.0f : 256.0f;
#pragma unroll
          for (int n = 0; n < NB; ++n) {
            mine[row0 * TC + 4 * n + c] = acc[2 * n] * f;
            mine[row1 * TC + 4 * n + c] = acc[2 * n + 1] * f;
          }
        }
        if constexpr (Q4K) {
          __syncwarp();
#pragma unroll
          for (int m = 0; m < S::TOKENS; ++m) {
            const float v = macc[m] + __shfl_xor_sync(0xffffffffu, macc[m], 16);
            if (lane < 16 && m < a.M) mine[lane * TC + (WIDE ? m : 2 * m + 1)] += v;
          }
        }
        __syncthreads();  // and the other buffer's readers are done before it is written again
        for (int x = threadIdx.x; x < outs; x += S::THREADS) {
          const int m = x / (16 * WR), r = x - m * 16 * WR;
          const int64_t n = n_super + r;
          const float* part = red + ((buf * S::WARPS + (r >> 4) * WK) * 16 + (r & 15)) * TC;
          float v = 0.0f;
          for (int w = 0; w < WK; ++w) {
            if constexpr (WIDE) {
              v += part[w * 16 * TC + m];
            } else {
              const float2 d = *reinterpret_cast<const float2*>(part + w * 16 * TC + 2 * m);
              v += d.x + d.y;
            }
          }
          if (n >= a.N) continue;
          if (CLUSTER || p.chunks > 1) {
            float* slot = acc_s + (i - g0) * outs + x;
            if (chunk > 0) v += *slot;
            *slot = v;
            if (CLUSTER || chunk < p.chunks - 1) continue;
          }
          const bool first = x == static_cast<int>(threadIdx.x);
          if (a.bias) v = __fadd_rn(v, first ? bias_first : __ldg(a.bias + n));
          if (a.resid) {
            if (a.gate) v = __fmul_rn(v, first ? gate_first : __ldg(a.gate + n));
            v = __fadd_rn(first ? resid_first : a.resid[m * a.ldr + n], v);
          }
          a.y[m * a.ldy + n] = v;
        }
        buf ^= 1;
      }
    }
    if constexpr (CLUSTER) {  // the sums of the cluster, in the order of its CTAs, which share out the outputs
      asm volatile("barrier.cluster.arrive.release;\nbarrier.cluster.wait.acquire;" ::: "memory");
      const int n_here = (min(own, g0 + group_n) - g0) * outs;
      for (int x = rank * S::THREADS + threadIdx.x; x < n_here; x += ranks * S::THREADS) {
        const int i = x / outs, y = x - i * outs, m = y / (16 * WR);
        const int64_t n = (cid + static_cast<int64_t>(g0 + i) * clusters) * WR * 16 + (y - m * 16 * WR);
        if (n >= a.N) continue;
        const float bias = a.bias ? __ldg(a.bias + n) : 0.0f, gate = a.gate ? __ldg(a.gate + n) : 1.0f;
        const float resid = a.resid ? a.resid[m * a.ldr + n] : 0.0f;
        float v = 0.0f;
#pragma unroll
        for (int r = 0; r < kMvRanks; ++r)
          if (r < ranks) v += mv_peer(smem_u32(acc_s + x), r);
        if (a.bias) v = __fadd_rn(v, bias);
        if (a.resid) {
          if (a.gate) v = __fmul_rn(v, gate);
          v = __fadd_rn(resid, v);
        }
        a.y[m * a.ldy + n] = v;
      }
      // none may go on while others read from it
      asm volatile("barrier.cluster.arrive.release;\nbarrier.cluster.wait.acquire;" ::: "memory");
    }
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");
}

template <bool Q4K, int NT, int XT>
cudaError_t launch_mv(const MulVecArgs& a, int num_sms, cudaStream_t s) {
  using S = MvShape<NT>;
  auto kern = mul_vec_kernel<Q4K, NT, XT, false>;
  auto kern_cl = mul_vec_kernel<Q4K, NT, XT, true>;
  cudaLaunchConfig_t cfg{};
  cfg.blockDim = dim3(S::THREADS);
  cfg.dynamicSmemBytes = kMvSmem;
  cfg.stream = s;
  cudaLaunchAttribute cluster{};
  cluster.id = cudaLaunchAttributeClusterDimension;
  cluster.val.clusterDim.x = cluster.val.clusterDim.y = cluster.val.clusterDim.z = 1;
  cfg.attrs = &cluster;
  cfg.numAttrs = 1;
  // Clusters of 1, 2, 4 and 8 CTAs that the device runs at a time (B200: 148, 74, 33, 15).
  static int fit[64][4] = {};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return cudaErrorInvalidDevice;
  if (fit[dev][0] == 0) {
    cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kMvSmem);
    if (e == cudaSuccess) e = cudaFuncSetAttribute(kern_cl, cudaFuncAttributeMaxDynamicSharedMemorySize, kMvSmem);
    if (e != cudaSuccess) return e;
    for (int c = 3; c >= 0; --c) {
      int n = num_sms;
      cfg.gridDim = dim3(num_sms << c);
      cluster.val.clusterDim.x = 1 << c;
      if (c > 0 && cudaOccupancyMaxActiveClusters(&n, kern_cl, &cfg) != cudaSuccess) {
        cudaGetLastError();
        n = 0;
      }
      fit[dev][c] = n;
    }
  }

  MvPlan p{};
  p.units = static_cast<int>((a.K + kMvUnitK - 1) / kMvUnitK);
  // Shared memory per unit: the digits, and per block s and the sum.
  const int per_unit = a.M * (3 * kMvUnitK + (Q4K ? 64 : 32));
  const int most = (S::X - a.M * (3 * 64 + 32)) / per_unit;
  // The CTAs of a cluster (2^c) that share out K, the warps of a CTA that share a tile's
  // units (WK) and the tiles side by side (WR): what finishes first when the super-tiles
  // go round the clusters that run at a time; the larger of equals, which spreads few
  // rows over more SMs.  In units' time with all warps at work (0.6 of it and less work,
  // with fewer: latency), fitted to 39 sizes x 4 clusters x 8 WK, of which it takes 0.7%
  // more than the best: a tile's end costs 0.5, a round of activation blocks 0.15, a
  // cluster's first join 0.5 and a later one 0.7.  One CTA, and clusters of 2, 4 and 8 with their best WK, us:
  //   6144 x 1024 Q4_0, 1 token 4.6, 5.8, 6.0, -; 8192 x 4096 Q4_0, 4 tokens 12.3, 12.0, 12.2, 16.3;
  //   49152 x 8192 Q4_K, 1 token 50, 53, 63, 86; 200 x 16384 Q4_0, 8 tokens 44, -, -, 8.5.
  // WK 1, 2, 4, 8 of one CTA: 49152 x 8192 Q4_K, 1 token 50.9, 50.7, 55.1, 54.1 us; 8192 x 4096
  // Q4_0, 4 tokens 15.5, 13.3, 12.4, 13.3; 6144 x 1024 Q4_0, 1 token 5.4, 4.8, 4.6, 4.6.
  const int tiles = static_cast<int>((a.N + 15) / 16);
  const auto over = [](int x, int y) { return (x + y - 1) / y; };
  float best = 0.0f;
  for (int c = 0; c <= 3; ++c) {
    const int per = (p.units + (1 << c) - 1) >> c, chunks = over(per, most);
    // Activations of one round are not worth sharing out (nor the host's time to weigh it).
    if (c > 0 && p.units * 8 * a.M <= S::THREADS / 8) break;
    // (a rank without units, or with fewer chunks than another, is not provided for)
    if (c > 0 && (fit[dev][c] == 0 || p.units < 1 << c || chunks > 1)) continue;
    const float stage = 0.15f * static_cast<float>((static_cast<int64_t>(per) * 8 * a.M + S::THREADS / 8 - 1) / (S::THREADS / 8));
    for (const int wk : {1, 2, 3, 4, 6, 8, 12}) {
      if (wk > S::WARPS / 2) break;
      // as few tiles side by side as the same number of rounds allows: they reach more SMs
      const int rounds = over(over(tiles, S::WARPS / wk), fit[dev][c]);
      const int wr = over(tiles, rounds * fit[dev][c]);
      const float busy = std::max(0.6f, static_cast<float>(wk * wr) / S::WARPS);
      const float join = c == 0 ? 0.0f : 0.7f * over(rounds, S::TILES / wr) - 0.2f;
      const float cost = rounds * (busy * over(per, wk) + 0.5f * chunks) + stage + join;
      if (best == 0.0f || cost <= best) {
        best = cost;
        p.wk = wk;
        p.wr = wr;
        p.rank_shift = c;
        p.chunk_units = over(per, chunks);
        p.chunks = over(per, p.chunk_units);
      }
    }
  }
  p.wk_inv = (65536 + p.wk - 1) / p.wk;
  p.supers = over(tiles, p.wr);
  p.pitch = p.chunk_units * kMvUnitK + 64;
  const uintptr_t xa = reinterpret_cast<uintptr_t>(a.x);
  p.vec = XT == kXF32 ? (xa % 16 == 0 && a.ldx % 4 == 0) : (xa % 8 == 0 && a.ldx % 4 == 0);
  const int clusters = std::min(p.supers, fit[dev][p.rank_shift]);
  if (p.rank_shift == 0) {
    kern<<<static_cast<unsigned>(clusters), S::THREADS, kMvSmem, s>>>(a, p);
    return cudaGetLastError();
  }
  cfg.gridDim = dim3(static_cast<unsigned>(clusters << p.rank_shift));
  cluster.val.clusterDim.x = 1u << p.rank_shift;
  return cudaLaunchKernelEx(&cfg, kern_cl, a, p);
}

}  // namespace

cudaError_t launch_mul_vec(const MulVecArgs& a, bool q4k, int xt, int num_sms, cudaStream_t s) {
#define B2Q_MV(Q, N)                                                                     \
  (xt == kXF32 ? launch_mv<Q, N, kXF32>(a, num_sms, s)                                   \
               : xt == kXF16 ? launch_mv<Q, N, kXF16>(a, num_sms, s) : launch_mv<Q, N, kXBF16>(a, num_sms, s))
  if (q4k) return a.M <= 2 ? B2Q_MV(true, 1) : a.M <= 4 ? B2Q_MV(true, 2) : B2Q_MV(true, 3);
  return a.M <= 2 ? B2Q_MV(false, 1) : a.M <= 4 ? B2Q_MV(false, 2) : B2Q_MV(false, 3);
#undef B2Q_MV
}

}  // namespace b2q
