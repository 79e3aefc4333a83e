// b2q_mul_mat_id_rows.cu -- the products of b2q_mul_mat_id with 4-bit weights
// (Q4_0) where the experts have few rows each (a decoding step): bound by the
// weights' bytes, 0.5625 a value, which are streamed once, as they are stored.
//
// A tile is 16 weight rows of one expert (with GLU 8 gate rows and the 8 up rows
// of the same outputs) against up to 32 of its slots.  All experts' tiles are
// numbered one after another and shared out evenly: every CTA (one per SM) has
// one run of them, so it seldom deals with more than two experts, whose rows
// of x it keeps in shared memory.  A warp has a tile to itself over all of K: no
// sums to join, and its own ring of cp.async chunks (16 rows x 256 values), which
// runs on from one tile into the next.
//
// Products are m16n8k16 with the weights as A.  K is taken in an order that suits
// the loads: lane t of a quad has the 8 codes of word t of a block, and x lies
// in shared memory in the same order, so that one 16-byte load feeds two products.
// Codes become q - 8 in fp16, which is exact; a block's sums are scaled by d and
// added in fp32, so a weight's value is never rounded.
//
// Measured: 24 tokens x 6 of 64 experts, 1408 -> 2048: 34 us for 87 MB; 8 of them until
// the first products (plan, first rows of x), 16 if nothing were computed, and the
// rest issue slots (8 warps an SM 35, 14 and 16 with shorter rings 33 to 36).
#include "b2q_groups.cuh"
#include "b2q_internal.h"

#include <algorithm>

namespace b2q {

namespace {

constexpr int kWarps = 12, kThreads = kWarps * 32;
constexpr int kRing = 5;                      // chunks of a warp
constexpr int kChunk = 16 * 128;              // bytes of weights
constexpr int kScales = 8 * 64;               // Q4_0: fp16 scales of 8 blocks
constexpr int kMaxNT = 4;                     // 8-slot tiles of a product
constexpr int kSmemMax = 227 * 1024;

constexpr int kChunkK = 256;
constexpr int kSlot = kChunk + kScales;
constexpr int kRingBytes = kWarps * kRing * kSlot;
constexpr int kPreBytes = (static_cast<int>(kMaxGroups) + 2) * 4 + 8;
constexpr int kFixed = (kRingBytes + kPreBytes + kMaxNT * 8 * 4 + kWarps * 4 + 127) & ~127;
static_assert(kSlot % 128 == 0, "a chunk's places are found by changing bits of its address");

// Bytes of a slot's row of x in shared memory: whole chunks, and 64 more, so that
// the rows of a quad's neighbours lie in other banks.
__host__ __device__ constexpr int64_t x_pitch(int64_t K) { return (K + kChunkK - 1) / kChunkK * kChunkK * 2 + 64; }

// 8-slot tiles of x's rows that a launch has shared memory for; 0: rows of K do not fit.
constexpr int launch_tiles(int64_t K) {
  const int64_t fit = (kSmemMax - kFixed) / (8 * x_pitch(K));
  return static_cast<int>(fit < kMaxNT ? fit : kMaxNT);
}
// 8-slot tiles that a run with slots for nt of them multiplies, and so reads: no more than there are rows for.
constexpr int product_tiles(int nt) { return nt; }
constexpr bool products_stay_inside() {
  for (int64_t K = 32; launch_tiles(K) > 0; K += 32)
    for (int nt = 1; nt <= launch_tiles(K); ++nt) {
      const int64_t last_row = product_tiles(nt) * 8 - 1, values = (K + kChunkK - 1) / kChunkK * kChunkK;
      if (last_row * x_pitch(K) + values * 2 > launch_tiles(K) * 8 * x_pitch(K)) return false;
    }
  return true;
}
static_assert(products_stay_inside(), "a product reads rows of x behind those that there is shared memory for");

__device__ __forceinline__ void mma16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, float c0, float c1,
                                      float c2, float c3) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};"
               : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(c0), "f"(c1), "f"(c2), "f"(c3));
}

__device__ __forceinline__ uint4 lds128(uint32_t a) {
  uint4 v;
  asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a));
  return v;
}
__device__ __forceinline__ uint32_t lds32(uint32_t a) {
  uint32_t v;
  asm volatile("ld.shared.b32 %0, [%1];" : "=r"(v) : "r"(a));
  return v;
}
__device__ __forceinline__ float lds_half(uint32_t a) {
  uint16_t v;
  asm volatile("ld.shared.u16 %0, [%1];" : "=h"(v) : "r"(a));
  return __half2float(__ushort_as_half(v));
}

// 8 codes of a Q4_0 word -> q - 8 as fp16 pairs: values (0, 2), (1, 3) of the
// low nibbles' four, then of the high ones'.  0x6400 | q is 1024 + q.
__device__ __forceinline__ uint32_t pick(uint32_t w, uint32_t mask) {
  uint32_t r;
  asm("lop3.b32 %0, %1, %2, %3, 0xea;" : "=r"(r) : "r"(w), "r"(mask), "r"(0x64006400u));  // (w & mask) | 0x6400..
  return r;
}
__device__ __forceinline__ void codes8(uint32_t w, uint32_t (&v)[4]) {
  const __half2 off = __half2half2(__ushort_as_half(0x6408));       // 1032
  const __half2 s16 = __half2half2(__ushort_as_half(0x2c00));       // 1 / 16
  const __half2 off16 = __half2half2(__ushort_as_half(0xd480));     // -72
  const uint32_t u = w >> 8;
  uint32_t p[4] = {pick(w, 0x000f000fu), pick(u, 0x000f000fu), pick(w, 0x00f000f0u), pick(u, 0x00f000f0u)};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __half2 h = *reinterpret_cast<const __half2*>(&p[i]);
    const __half2 r = i < 2 ? __hsub2(h, off) : __hfma2(h, s16, off16);
    v[i] = *reinterpret_cast<const uint32_t*>(&r);
  }
}

struct RowsTile {
  int e;           // expert
  int row;         // first output row
  int begin, end;  // sorted slots
};

template <bool GLU, bool OUT32>
__global__ void __launch_bounds__(kThreads, 1) id_rows_kernel(const MulMatIdArgs p, const int tile_slots) {
  constexpr int OT = OUT32 ? 0 : 1;
  using OV = typename Val<OT>::type;
  constexpr int ROWS = GLU ? 8 : 16;  // outputs of a tile
  extern __shared__ __align__(1024) uint8_t smem[];
  uint8_t* ring = smem;
  int* pre = reinterpret_cast<int*>(smem + kRingBytes);
  int* slots = reinterpret_cast<int*>(smem + kRingBytes + kPreBytes);
  int* warp_sums = slots + kMaxNT * 8;
  uint8_t* xs = smem + kFixed;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int g = lane >> 2, q = lane & 3;
  const int r_tiles = static_cast<int>((p.n + ROWS - 1) / ROWS);
  const int pitch = static_cast<int>(x_pitch(p.K));

  grid_wait();
  // pre[e]: tiles of the experts before e.
  int carry = 0;
  for (int e0 = 0; e0 <= p.E; e0 += kThreads) {
    const int e = e0 + threadIdx.x;
    int n = 0;
    if (e < p.E) {
      const int b = group_begin(p.offsets, e, p.S);
      n = (group_end(p.offsets, e, p.E, p.S, b) - b + tile_slots - 1) / tile_slots * r_tiles;
    }
    int inc = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int u = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += u;
    }
    if (lane == 31) warp_sums[warp] = inc;
    __syncthreads();
    int before = carry;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      if (w < warp) before += warp_sums[w];
      carry += warp_sums[w];
    }
    if (e <= p.E) pre[e] = before + inc - n;
    __syncthreads();
  }
  const int total = max(0, pre[p.E]);
  const int t0 = static_cast<int>(static_cast<int64_t>(total) * blockIdx.x / gridDim.x);
  const int t1 = static_cast<int>(static_cast<int64_t>(total) * (blockIdx.x + 1) / gridDim.x);

  // The run that tile t belongs to: one expert's tiles against the same slots.
  auto run_of = [&](int t, RowsTile& r, int& first, int& last) {
    int lo = 0, hi = p.E;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (pre[mid] <= t) lo = mid;
      else hi = mid;
    }
    const int part = (t - pre[lo]) / r_tiles;
    const int begin = group_begin(p.offsets, lo, p.S);
    const int end = group_end(p.offsets, lo, p.E, p.S, begin);
    r.e = lo;
    r.begin = max(0, min(end, begin + part * tile_slots));
    r.end = min(end, r.begin + tile_slots);
    first = pre[lo] + part * r_tiles;  // its tile 0
    last = min(t1, first + r_tiles);
  };

  const int chunks = static_cast<int>((p.K + kChunkK - 1) / kChunkK);
  const int row_bytes = static_cast<int>(p.K / 2);
  // What the warp asks for next: chunk `ic` of tile `it` in the run [ifirst, ilast).
  RowsTile ir{};
  int it = t0, ifirst = 0, ilast = t0, ic = 0;
  const uint8_t* isrc[4];
  bool ithere[4];
  const uint16_t* iscale = nullptr;
  auto next_tile = [&](int& t, RowsTile& r, int& first, int& last, int start) {
    // the warp's next tile at or after `start`, entering the next runs as needed
    t = start;
    while (t >= last && last < t1) {
      run_of(last, r, first, last);
      t = max(first, t0) + warp;  // (runs are entered at their first tile, or at the CTA's)
    }
    if (t < last) r.row = (t - first) * ROWS;
  };
  auto aim = [&]() {  // addresses of tile `it`
    if (it >= t1) return;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int r = (lane >> 3) + 4 * i;  // weight row of the tile
      const int out = GLU ? ir.row + (r & 7) : ir.row + r;
      ithere[i] = out < p.n;
      const int64_t row = (GLU && r >= 8 ? p.n : 0) + (ithere[i] ? out : 0);
      isrc[i] = static_cast<const uint8_t*>(p.w) + (static_cast<int64_t>(ir.e) * p.rows + row) * row_bytes + (lane & 7) * 16;
    }
    // lane: block lane / 4 of the chunk, and 8 of its scales from a multiple of 8 rows on
    const int64_t first = static_cast<int64_t>(ir.e) * p.rows + ir.row + (GLU && (lane & 2) ? p.n : 0);
    const int64_t at = (first & ~int64_t{7}) + (GLU ? (lane & 1) * 8 : q * 8);
    iscale = at < p.lds ? p.scales + at + g * p.lds : nullptr;
  };
  const uint32_t ring32 = static_cast<uint32_t>(__cvta_generic_to_shared(ring)) + warp * kRing * kSlot;
  // A block's place goes by the row: rows 0, 4, 8 and 12 below a lane's.
  const int arow = lane >> 3, ac = lane & 7;
  const uint32_t place0 = arow * 128 + (ac ^ arow) * 16, place1 = (arow + 4) * 128 + (ac ^ (arow + 4)) * 16;
  uint32_t put = ring32, take = ring32;
  const uint32_t ring_end = ring32 + kRing * kSlot;
  auto ask = [&]() {  // the next chunk, or an empty group when all are asked for
    if (it < t1) {
      const bool in = ic * 128 + ac * 16 < row_bytes;
      cp16(put + place0, isrc[0], in && ithere[0]);
      cp16(put + place1, isrc[1], in && ithere[1]);
      cp16(put + place0 + 1024, isrc[2], in && ithere[2]);
      cp16(put + place1 + 1024, isrc[3], in && ithere[3]);
      const bool there = iscale && (ic * 8 + g) * 32 < p.K && (GLU || q < 3);
      cp16(put + kChunk + g * 64 + q * 16, there ? iscale : p.scales, there);
      if (iscale) iscale += 8 * p.lds;
      if (++ic == chunks) {
        ic = 0;
        next_tile(it, ir, ifirst, ilast, it + kWarps);
        aim();
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) isrc[i] += 128;
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
    put = put + kSlot == ring_end ? ring32 : put + kSlot;
  };
  next_tile(it, ir, ifirst, ilast, t0);
  if (it >= ilast) it = t1;  // nothing for this warp
  aim();
  for (int i = 0; i < kRing - 1; ++i) ask();

  // The warp's tiles from, from + kWarps, ... of a run against NT times 8 slots.
  const uint32_t xb = static_cast<uint32_t>(__cvta_generic_to_shared(xs)) + g * pitch + q * 16;
  auto tiles_of = [&](auto nt_c, RowsTile& r, int first, int from, int last) {
    constexpr int NT = decltype(nt_c)::value;
    for (int t = from; t < last; t += kWarps) {
      r.row = (t - first) * ROWS;
      float acc[NT][4] = {};
      // where a lane's two rows' scales lie
      const int64_t f = static_cast<int64_t>(r.e) * p.rows + r.row;
      const uint32_t sa = kChunk + (static_cast<int>(f & 7) + g) * 2;
      const uint32_t sb = GLU ? kChunk + 32 + (static_cast<int>((f + p.n) & 7) + g) * 2 : sa + 16;
      uint32_t xc = xb;
      for (int c = 0; c < chunks; ++c) {
        asm volatile("cp.async.wait_group %0;" ::"n"(kRing - 2) : "memory");
        __syncwarp();
        const uint32_t row = take + g * 128 + (g << 4) + q * 4;  // block b: with b << 4 added without carry
        const int blocks = min(8, static_cast<int>(p.K / 32) - c * 8);
        auto block = [&](int b) {
          uint32_t lo[4], hi[4];
          const uint32_t at = row ^ (b << 4);
          codes8(lds32(at), lo);
          codes8(lds32(at + 1024), hi);
          const float da = lds_half(take + sa + b * 64), db = lds_half(take + sb + b * 64);
          const uint32_t a0[4] = {lo[0], hi[0], lo[1], hi[1]}, a1[4] = {lo[2], hi[2], lo[3], hi[3]};
#pragma unroll
          for (int j = 0; j < NT; ++j) {
            const uint4 x = lds128(xc + j * 8 * pitch + b * 64);
            float d[4], e[4];
            mma16(e, a0, x.x, x.y, 0.0f, 0.0f, 0.0f, 0.0f);
            mma16(d, a1, x.z, x.w, e[0], e[1], e[2], e[3]);
            acc[j][0] = fmaf(da, d[0], acc[j][0]);
            acc[j][1] = fmaf(da, d[1], acc[j][1]);
            acc[j][2] = fmaf(db, d[2], acc[j][2]);
            acc[j][3] = fmaf(db, d[3], acc[j][3]);
          }
        };
        if (blocks == 8) {
#pragma unroll
          for (int b = 0; b < 8; ++b) block(b);
        } else {
          for (int b = 0; b < blocks; ++b) block(b);
        }
        xc += kChunkK * 2;
        take = take + kSlot == ring_end ? ring32 : take + kSlot;
        __syncwarp();  // all lanes have read the chunk whose place the next one takes
        ask();
      }
      // The tile's outputs: a lane has rows g and g + 8 (GLU: gate and up of row g) of slots 2 q and 2 q + 1.
      const int row = r.row + g;
      const float* bias = p.bias ? p.bias + static_cast<int64_t>(r.e) * p.rows : nullptr;
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int s = slots[j * 8 + 2 * q + i];
          if (s < 0) continue;
          OV* out = static_cast<OV*>(p.y) + s * p.ldy;
          if constexpr (GLU) {
            if (row < p.n) {
              const float gate = acc[j][i] + (bias ? __ldg(bias + row) : 0.0f);
              const float lin = acc[j][2 + i] + (bias ? __ldg(bias + p.n + row) : 0.0f);
              out[row] = Val<OT>::to(gate / (1.0f + expf(-gate)) * lin);
            }
          } else {
            if (row < p.n) out[row] = Val<OT>::to(acc[j][i] + (bias ? __ldg(bias + row) : 0.0f));
            if (row + 8 < p.n) out[row + 8] = Val<OT>::to(acc[j][2 + i] + (bias ? __ldg(bias + row + 8) : 0.0f));
          }
        }
    }
  };

  RowsTile r{};
  int first = 0, last = t0;
  while (last < t1) {  // run after run
    const int start = last;
    run_of(start, r, first, last);
    __syncthreads();  // the rows of the run before are no longer read
    const int count = r.end - r.begin, nt = (count + 7) / 8;
    for (int i = threadIdx.x; i < kMaxNT * 8; i += kThreads) {
      int s = -1;
      if (i < count) {
        s = __ldg(p.order + r.begin + i);
        if (s < 0 || s >= p.S) s = -1;
      }
      slots[i] = s;
    }
    __syncthreads();
    // x rows: 16 bytes a thread, zeros behind the row's end and for the missing slots of the last 8
    const int vecs = (pitch - 64) / 16;
    for (int i = threadIdx.x; i < nt * 8 * vecs; i += kThreads) {
      const int m = i / vecs, j = i - m * vecs;
      uint4 v = make_uint4(0, 0, 0, 0);
      const int s = slots[m];
      if (s >= 0 && static_cast<int64_t>(j) * 8 < p.K)
        v = __ldg(reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p.x) + (s / p.per_row) * p.ldx) + j);
      uint8_t* row = xs + m * pitch;
      // two groups of 4 of a block, each as values 0, 2, 1, 3
      const int group = (2 * j) & 7;
      uint8_t* b = row + (j >> 2) * 64;
      *reinterpret_cast<uint2*>(b + (group & 3) * 16 + (group >> 2) * 8) =
          make_uint2(__byte_perm(v.x, v.y, 0x5410), __byte_perm(v.x, v.y, 0x7632));
      *reinterpret_cast<uint2*>(b + ((group + 1) & 3) * 16 + (group >> 2) * 8) =
          make_uint2(__byte_perm(v.z, v.w, 0x5410), __byte_perm(v.z, v.w, 0x7632));
    }
    __syncthreads();
    const int from = start + warp;
    if (nt <= 1) tiles_of(std::integral_constant<int, product_tiles(1)>(), r, first, from, last);
    else if (nt == 2) tiles_of(std::integral_constant<int, product_tiles(2)>(), r, first, from, last);
    else if (nt == 3) tiles_of(std::integral_constant<int, product_tiles(3)>(), r, first, from, last);
    else tiles_of(std::integral_constant<int, product_tiles(kMaxNT)>(), r, first, from, last);
  }
  asm volatile("cp.async.wait_all;" ::: "memory");
  // Slots of no group: rows of zeros.
  const int none = group_begin(p.offsets, p.E, p.S);
  for (int64_t i = none + static_cast<int64_t>(blockIdx.x) * kWarps + warp; i < p.S;
       i += static_cast<int64_t>(gridDim.x) * kWarps) {
    const int s = __ldg(p.order + i);
    if (s < 0 || s >= p.S) continue;
    OV* out = static_cast<OV*>(p.y) + s * p.ldy;
    for (int64_t j = lane; j < p.n; j += 32) out[j] = Val<OT>::to(0.0f);
  }
}

template <bool GLU, bool OUT32>
cudaError_t launch_shape(const MulMatIdArgs& a, int num_sms, cudaStream_t s) {
  const int64_t pitch = x_pitch(a.K);
  const int nt = launch_tiles(a.K);
  if (nt < 1) return cudaErrorInvalidValue;
  constexpr auto k = id_rows_kernel<GLU, OUT32>;
  if (cudaError_t e = allow_smem<k>(kSmemMax)) return e;
  return launch_early(k, dim3(static_cast<unsigned>(num_sms)), dim3(kThreads), kFixed + nt * 8 * pitch, s, 1, a, nt * 8);
}

}  // namespace

bool id_rows_fits(int64_t K) { return launch_tiles(K) > 0; }

cudaError_t launch_id_rows(const MulMatIdArgs& a, int ytype, int num_sms, cudaStream_t s) {
  const bool out32 = ytype == kXF32;
  return a.glu ? (out32 ? launch_shape<true, true>(a, num_sms, s) : launch_shape<true, false>(a, num_sms, s))
               : (out32 ? launch_shape<false, true>(a, num_sms, s) : launch_shape<false, false>(a, num_sms, s));
}

}  // namespace b2q
