// b2q_mul_mat_id.cu -- matrix products whose weight goes by row: slot s of a
// plan multiplies the weight of its expert,
//   y[s][r] = sum_k W[e(s)][r][k] x[s / per_row][k] (+ bias[e][r]),
// or, with GLU, silu(y[s][r]) * y[s][n + r] of a weight of 2 n rows.
//
// One kernel for every number of rows.  Weight rows are the M of the MMA (256
// over a pair of CTAs, cta_group::2), a group's sorted slots its N, in tiles of
// up to 256 whose width goes by the group: a group of 3 rows costs an N of 32, so
// a decoding step streams each used weight once at the rate of the memory, and
// a prompt's groups run at the tensor cores' rate.  The pairs are persistent and
// find their tiles themselves from the plan's offsets, so that the host never
// learns the groups' sizes.
//   A   weight tile by TMA, one box a stage: with GLU 64 gate rows and the 64 up
//       rows that belong to them, so both sums of an output end in one CTA
//   B   rows of x by their numbers, cp.async into the layout of the MMA; a thread
//       of its own waits for them, makes them visible to the tensor core and
//       reports them to the pair's leader: no sorted copy of x is written or read
//   D   fp32 in tensor memory, two accumulators of 256 columns; the epilogue
//       scatters rows to their slots
// 4-bit weights (Q4_0): the nibble blocks come by TMA, 256 values of a row at a
// time, and eight warps widen them into A.  A weight (q - 8) d has up to 15 bits,
// so d is taken as a number of 7 bits and one of 4, whose products with q - 8 are
// exact in fp16, and two MMAs add up to the weight as it is (|8 d| < 65504).
// Few rows with such weights go to b2q_mul_mat_id_rows.cu.
//
// Measured: gate and up of 8192 tokens x 4 of 32 experts, 2048 -> 1408, bf16: 326 us alone,
// 1160 TFLOP/s, tensor pipe 63% active; 388, 975 TFLOP/s, in calls that follow one
// another for seconds, where the power cap holds the clocks down (TMA gathers of 4 rows instead of cp.async 946,
// a sorted copy of x and TMA boxes 353); of 40 tokens x 4 of 64 experts, 2048 -> 1024:
// 77 us, 5790 GB/s; one token x 6 experts, 2048 -> 1408: 20 us, 3400 GB/s, a third of it
// set-up.
#include "b2q_groups.cuh"
#include "b2q_internal.h"
#include "b2q_ptx.cuh"

#include <algorithm>
#include <atomic>

namespace b2q {

namespace {

__device__ unsigned int g_id_status = 0;

constexpr int kBM = 128;              // weight rows per CTA (256 per pair)
constexpr int kBN = 256;              // slots per tile, at most
constexpr int kStageK = 64;           // values of K per stage: 128 bytes
constexpr int kABytes = kBM * kStageK * 2;
constexpr int kBBytes = kBN / 2 * kStageK * 2;
constexpr int kAccs = 2;
// Rows per expert, on average, up to which the rows kernel does 4-bit weights.  Measured over 21 shapes (8, 32 and 128
// experts, K 256 to 4096, 512 to 2816 weight rows, cold weights), rows kernel over this one: 0.72 of the time with 8 rows an
// expert (0.48 to 0.96), 0.82 with 12 (0.57 to 1.09), 0.89 with 16 (0.65 to 1.19), 1.00 with 24 (0.79 to 1.31).  With 16
// it loses where this kernel's tiles just fill their waves or leave most pairs idle anyway: 32 and 8 experts of gate and
// up 1024 -> 512 28.6 us against 25.0 and 18.2 against 15.3, 512 -> 512 18.8 against 18.1, 8 experts of 1408 -> 2048 20.4
// against 18.9; and gains 66.5 against 84.8 (32 experts, 2048 -> 1408), 41.8 against 52.5 (1408 -> 2048), 62 against 82 (128
// of 512 -> 2048).
constexpr int kFewRows = 16;
// Q4_0: a raw slot is 256 values of the CTA's 128 rows: nibbles in two boxes of
// 64 rows, and each box's fp16 scales from the multiple of 8 rows below its first
// (a TMA copy starts on 16 bytes).
constexpr int kRawK = 256;
constexpr int kRawBox = 64 * kRawK / 2, kScaleCols = 72, kScaleBox = kRawK / 32 * kScaleCols * 2;
constexpr int kRawBytes = 2 * kRawBox + 2 * kScaleBox;
constexpr int kRawStride = (kRawBytes + 1023) / 1024 * 1024;
static_assert(kScaleBox % 128 == 0, "TMA destinations");

template <int W, bool GLU>
struct IdShape {
  static constexpr bool Q4 = W == kWQ4;
  // Stages of A and of B have rings of their own: B's rows take longer to come.
  static constexpr int AS = Q4 ? 3 : 5, BS = Q4 ? 4 : 7, RAWS = Q4 ? 2 : 0;
  static constexpr int A = Q4 ? 2 * kABytes : kABytes;  // 4 bits: the weights as sums of two numbers
  static constexpr int OFF_B = AS * A;
  static constexpr int EPI = Q4 ? 8 : 16;   // epilogue warps
  static constexpr int CONV = Q4 ? 8 : 0;   // widening warps
  static constexpr int GATHER = 4;          // warps that fetch rows of x
  static constexpr int WARPS = 2 + EPI + CONV + GATHER + 1, THREADS = WARPS * 32;
  static constexpr int CHUNK = GLU ? 16 : 32;  // accumulator columns that an epilogue warp has in registers
  static constexpr int OFF_RAW = OFF_B + BS * kBBytes;
  static constexpr int OFF_SWAP = OFF_RAW + RAWS * kRawStride;
  static constexpr int SWAP = GLU ? EPI * 32 * 8 * 4 : 0;
  static constexpr int OFF_PRE = OFF_SWAP + SWAP;
  static constexpr int OFF_BARS = OFF_PRE + (static_cast<int>(kMaxGroups) + 2) * 4 + 8;
  static constexpr int NBARS = 2 * AS + 3 * BS + 2 * RAWS + 2 * kAccs + 1;
  static constexpr int SMEM = OFF_BARS + NBARS * 8 + 8 + 4 + 4 + 2 * EPI * 4 + THREADS / 32 * 4 + 1024;
};
static_assert(IdShape<1, true>::SMEM <= 227 * 1024 && IdShape<kWQ4, true>::SMEM <= 227 * 1024, "shared memory");
static_assert(IdShape<1, true>::OFF_BARS % 8 == 0 && IdShape<kWQ4, true>::OFF_BARS % 8 == 0, "barriers");

struct IdTile {
  int e;           // expert
  int r0, r1;      // first weight row of the CTA's two boxes, within the expert
  int n0;          // first output column of the CTA's first box
  int begin, end;  // sorted slots
  int width;       // N of the MMA: a multiple of 32
};

template <bool GLU>
__device__ __forceinline__ IdTile id_tile(const MulMatIdArgs& a, const int* pre, int tile, int w_tiles, int rank) {
  int lo = 0, hi = a.E;  // pre[lo] <= tile < pre[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (pre[mid] <= tile) lo = mid;
    else hi = mid;
  }
  IdTile t;
  t.e = lo;
  const int local = tile - pre[lo];
  const int wt = local % w_tiles, tt = local / w_tiles;
  const int begin = group_begin(a.offsets, lo, a.S);
  const int end = group_end(a.offsets, lo, a.E, a.S, begin);
  // (a plan that changes under the kernel, or whose groups overlap without end, still leads to some slots)
  const int parts = max(1, (end - begin + kBN - 1) / kBN);
  const int width = max(32, ((end - begin + parts - 1) / parts + 31) & ~31);
  t.begin = max(0, min(end, begin + tt * width));
  t.end = min(end, t.begin + width);
  t.width = max(32, min(width, (t.end - t.begin + 31) & ~31));
  t.n0 = GLU ? wt * kBM + rank * (kBM / 2) : wt * 2 * kBM + rank * kBM;
  t.r0 = t.n0;
  t.r1 = GLU ? static_cast<int>(a.n) + t.n0 : t.n0 + kBM / 2;
  return t;
}

struct IdMaps {
  CUtensorMap w, scales;
};

__device__ __forceinline__ uint32_t hsub2_u(uint32_t a, uint32_t b) {
  __half2 r = __hsub2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b));
  return *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ uint32_t hmul2_u(uint32_t a, uint32_t b) {
  __half2 r = __hmul2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b));
  return *reinterpret_cast<const uint32_t*>(&r);
}

// Four 4-bit codes in the low halves of four bytes -> q - 8, two fp16 pairs.
// 0x64 above a byte q is the fp16 number 1024 + q.
__device__ __forceinline__ uint2 codes4(uint32_t q) {
  uint32_t a, b;
  asm("prmt.b32 %0, %1, %2, 0x4140;" : "=r"(a) : "r"(q), "r"(0x64646464u));
  asm("prmt.b32 %0, %1, %2, 0x4342;" : "=r"(b) : "r"(q), "r"(0x64646464u));
  const uint32_t bias = 0x64086408u;  // 1032
  return make_uint2(hsub2_u(a, bias), hsub2_u(b, bias));
}

template <int W, bool GLU, bool OUT32>
__global__ void __launch_bounds__(IdShape<W, GLU>::THREADS, 1)
    mul_mat_id_kernel(const __grid_constant__ IdMaps maps, const MulMatIdArgs p) {
  using Sh = IdShape<W, GLU>;
  using OV = typename Val<OUT32 ? 0 : (W == 2 ? 2 : 1)>::type;
  constexpr int OT = OUT32 ? 0 : (W == 2 ? 2 : 1);
  constexpr bool Q4 = Sh::Q4;
  constexpr int AS = Sh::AS, BS = Sh::BS, RS = Sh::RAWS;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  uint8_t* raws = smem + Sh::OFF_RAW;
  float* swap = reinterpret_cast<float*>(smem + Sh::OFF_SWAP);
  int* pre = reinterpret_cast<int*>(smem + Sh::OFF_PRE);
  uint64_t* a_full = reinterpret_cast<uint64_t*>(smem + Sh::OFF_BARS);  // used in the leader, as b_full
  uint64_t* a_empty = a_full + AS;
  uint64_t* b_full = a_empty + AS;
  uint64_t* b_empty = b_full + BS;
  uint64_t* x_full = b_empty + BS;  // rows of x have arrived in this CTA
  uint64_t* raw_full = x_full + BS;
  uint64_t* raw_empty = raw_full + RS;
  uint64_t* acc_full = raw_empty + RS;
  uint64_t* acc_empty = acc_full + kAccs;  // used in the leader: both CTAs' epilogue warps
  uint64_t* mma_done = acc_empty + kAccs;
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(mma_done + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_holder + 1);
  volatile int* pair_ok = abort_flag + 1;       // [2][EPI]
  int* warp_sums = const_cast<int*>(pair_ok) + 2 * Sh::EPI;  // [WARPS]
  unsigned int* status = &g_id_status;
  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();
  const bool leader = rank == 0;
  const int cluster = blockIdx.x >> 1, nclusters = gridDim.x >> 1;
  const int w_tiles = static_cast<int>((p.n + (GLU ? kBM : 2 * kBM) - 1) / (GLU ? kBM : 2 * kBM));
  const int kst = static_cast<int>((p.K + kStageK - 1) / kStageK);

  if (threadIdx.x == 0) {
    for (int s = 0; s < AS; ++s) {
      mbar_init(&a_full[s], Q4 ? 8 : 1);  // four widening warps of each CTA, or the producer
      mbar_init(&a_empty[s], 1);
    }
    for (int s = 0; s < BS; ++s) {
      mbar_init(&b_full[s], 2);
      mbar_init(&b_empty[s], 1);
      mbar_init(&x_full[s], Sh::GATHER * 32);
    }
    for (int s = 0; s < RS; ++s) {
      mbar_init(&raw_full[s], 1);
      mbar_init(&raw_empty[s], Sh::CONV);
    }
    for (int a = 0; a < kAccs; ++a) {
      mbar_init(&acc_full[a], 1);
      mbar_init(&acc_empty[a], 2 * Sh::EPI);
    }
    mbar_init(mma_done, 1);
    *abort_flag = 0;
    fence_mbarrier_init();
    tma_prefetch_desc(&maps.w);
    if constexpr (Q4) tma_prefetch_desc(&maps.scales);
  }
  // (Tensor memory too is taken only now: the kernel before may still have blocks that ask for it.)
  grid_wait();
  if (warp == 1) {
    tmem_alloc_pair(tmem_holder, kAccs * kBN);
    tmem_relinquish_pair();
  }
  // pre[e]: tiles of the experts before e.  Two experts a thread.
  {
    int n[2] = {0, 0};
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int e = 2 * threadIdx.x + i;
      if (e < p.E) {
        const int b = group_begin(p.offsets, e, p.S);
        n[i] = (group_end(p.offsets, e, p.E, p.S, b) - b + kBN - 1) / kBN * w_tiles;
      }
    }
    int inc = n[0] + n[1];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int u = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += u;
    }
    if (lane == 31) warp_sums[warp] = inc;
    __syncthreads();
    int before = 0;
    for (int w = 0; w < warp; ++w) before += warp_sums[w];
    const int at = before + inc - n[0] - n[1];
    if (2 * threadIdx.x <= static_cast<unsigned>(p.E)) pre[2 * threadIdx.x] = at;
    if (2 * threadIdx.x + 1 <= static_cast<unsigned>(p.E)) pre[2 * threadIdx.x + 1] = at + n[0];
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync();  // both CTAs' barriers exist before any arrival crosses the pair
  tc_fence_after();
  const uint32_t tmem_base = *tmem_holder;
  const int num_tiles = pre[p.E];

  if (warp == 0) {
    // ------------------------------------- producer: the weights, as they are stored
    if (elect_one()) {
      if constexpr (!Q4) {
        const uint32_t full0 = cluster_addr(a_full, 0);
        uint32_t stage = 0, phase = 0, issued_mask = 0, issued_par = 0;
        bool ok = true;
        for (int tile = cluster; ok && tile < num_tiles; tile += nclusters) {
          const IdTile t = id_tile<GLU>(p, pre, tile, w_tiles, rank);
          for (int ks = 0; ks < kst; ++ks) {
            if (!mbar_wait(&a_empty[stage], phase ^ 1u, status, kDevWaitProducer, abort_flag)) {
              ok = false;
              break;
            }
            uint8_t* sb = smem + stage * Sh::A;
            const uint32_t fb = full0 + stage * 8;
            if (leader) mbar_arrive_expect_tx(&a_full[stage], 2 * kABytes);  // both CTAs' bytes
            tma_load_4d_pair(sb, &maps.w, fb, ks * kStageK, t.r0, 0, t.e);
            issued_mask |= 1u << stage;
            issued_par = (issued_par & ~(1u << stage)) | (phase << stage);
            if (++stage == AS) {
              stage = 0;
              phase ^= 1u;
            }
          }
        }
        if (leader)  // every issued copy of both CTAs lands before the pair may exit
          for (int s = 0; s < AS; ++s)
            if ((issued_mask >> s) & 1u) mbar_wait(&a_full[s], (issued_par >> s) & 1u, status, kDevWaitDrain, nullptr);
      } else {
        uint32_t raw = 0, phase = 0, issued_mask = 0, issued_par = 0;
        bool ok = true;
        for (int tile = cluster; ok && tile < num_tiles; tile += nclusters) {
          const IdTile t = id_tile<GLU>(p, pre, tile, w_tiles, rank);
          const int y0 = static_cast<int>(t.e * p.rows + t.r0), y1 = static_cast<int>(t.e * p.rows + t.r1);
          for (int rs = 0; rs * 4 < kst; ++rs) {
            if (!mbar_wait(&raw_empty[raw], phase ^ 1u, status, kDevWaitProducer, abort_flag)) {
              ok = false;
              break;
            }
            uint8_t* rb = raws + raw * kRawStride;
            mbar_arrive_expect_tx(&raw_full[raw], kRawBytes);
            tma_load_2d(rb, &maps.w, &raw_full[raw], rs * (kRawK / 2), y0);
            tma_load_2d(rb + kRawBox, &maps.w, &raw_full[raw], rs * (kRawK / 2), y1);
            tma_load_2d(rb + 2 * kRawBox, &maps.scales, &raw_full[raw], y0 & ~7, rs * (kRawK / 32));
            tma_load_2d(rb + 2 * kRawBox + kScaleBox, &maps.scales, &raw_full[raw], y1 & ~7, rs * (kRawK / 32));
            issued_mask |= 1u << raw;
            issued_par = (issued_par & ~(1u << raw)) | (phase << raw);
            if (++raw == RS) {
              raw = 0;
              phase ^= 1u;
            }
          }
        }
        for (int s = 0; s < RS; ++s)
          if ((issued_mask >> s) & 1u) mbar_wait(&raw_full[s], (issued_par >> s) & 1u, status, kDevWaitDrain, nullptr);
      }
    }
  } else if (warp == 1) {
    // ------------------------------------------------- MMA issuer (leader)
    if (leader && elect_one()) {
      uint32_t as = 0, aphase = 0, bs = 0, bphase = 0, n = 0;
      bool ok = true;
      for (int tile = cluster; ok && tile < num_tiles; tile += nclusters, ++n) {
        const IdTile t = id_tile<GLU>(p, pre, tile, w_tiles, rank);
        const uint32_t idesc = W == 2 ? idesc_bf16(2 * kBM, t.width) : idesc_f16(2 * kBM, t.width);
        const uint32_t a = n & (kAccs - 1), apar = (n / kAccs) & 1u;
        if (!mbar_wait_cluster(&acc_empty[a], apar ^ 1u, status, kDevWaitMma, abort_flag)) break;
        tc_fence_after();
        const uint32_t d = tmem_base + a * kBN;
        for (int ks = 0; ks < kst; ++ks) {
          if (!mbar_wait(&b_full[bs], bphase, status, kDevWaitMma, abort_flag) ||
              !mbar_wait(&a_full[as], aphase, status, kDevWaitMma, abort_flag)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t a_base = smem_u32(smem + as * Sh::A);
          const uint32_t b_base = smem_u32(smem + Sh::OFF_B + bs * kBBytes);
#pragma unroll
          for (int j = 0; j < kStageK / 16; ++j)
            mma_f16_pair(d, smem_desc_k_sw128(a_base + j * 32), smem_desc_k_sw128(b_base + j * 32), idesc,
                         (ks | j) != 0 ? 1u : 0u);
          if constexpr (Q4) {
#pragma unroll
            for (int j = 0; j < kStageK / 16; ++j)
              mma_f16_pair(d, smem_desc_k_sw128(a_base + kABytes + j * 32), smem_desc_k_sw128(b_base + j * 32), idesc, 1u);
          }
          mma_commit_pair(&a_empty[as], 0x3);
          mma_commit_pair(&b_empty[bs], 0x3);
          if (++as == AS) {
            as = 0;
            aphase ^= 1u;
          }
          if (++bs == BS) {
            bs = 0;
            bphase ^= 1u;
          }
        }
        if (ok) mma_commit_pair(&acc_full[a], 0x3);
      }
      mma_commit_pair(mma_done, 0x1);
      mbar_wait(mma_done, 0, status, kDevWaitDrain, nullptr);
    }
  } else if (warp < 2 + Sh::EPI) {
    // ------------------------------------------------------------ epilogue
    const int ew = warp - 2;
    const int quarter = warp & 3;  // TMEM lane quarter that this warp may access
    const int group = ew >> 2;
    constexpr int GROUPS = Sh::EPI / 4;
    const uint32_t tlane = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16);
    // GLU: quarters 0 and 1 hold gate sums, 2 and 3 the up sums of the same outputs.
    const bool up = GLU && quarter >= 2;
    const int bar = 1 + group * 2 + (quarter & 1);
    const int partner = 2 + group * 4 + (((quarter ^ 2) + 2) & 3) - 2;  // epilogue warp of the other quarter
    (void)bar;
    (void)partner;
    uint32_t n = 0;
    for (int tile = cluster; tile < num_tiles; tile += nclusters, ++n) {
      const IdTile t = id_tile<GLU>(p, pre, tile, w_tiles, rank);
      const uint32_t a = n & (kAccs - 1), apar = (n / kAccs) & 1u;
      const int row = GLU ? t.n0 + (quarter & 1) * 32 + lane : t.n0 + quarter * 32 + lane;
      const bool nv = row < p.n;
      float bias = 0.0f;
      if (p.bias && nv) bias = __ldg(p.bias + static_cast<int64_t>(t.e) * p.rows + (up ? p.n : 0) + row);
      bool ok = __all_sync(0xffffffffu, mbar_wait(&acc_full[a], apar, status, kDevWaitEpilogue, abort_flag));
      if constexpr (GLU) {  // both warps of an output go on, or none: neither may wait for the other alone
        if (lane == 0) pair_ok[(n & 1) * Sh::EPI + ew] = ok;
        asm volatile("bar.sync %0, 64;" ::"r"(bar) : "memory");
        ok = pair_ok[(n & 1) * Sh::EPI + ew] && pair_ok[(n & 1) * Sh::EPI + partner];
      }
      if (!ok) break;
      tc_fence_after();
      const uint32_t tacc = tlane + a * kBN;
      OV* out = static_cast<OV*>(p.y) + row;
      const int chunks = (t.width + Sh::CHUNK - 1) / Sh::CHUNK;
      bool released = false;
      for (int c = group; c < chunks; c += GROUPS) {
        uint32_t acc[Sh::CHUNK];
        if constexpr (Sh::CHUNK == 32) tmem_ld_32x32b_x32(tacc + c * 32, acc);
        else tmem_ld_32x32b_x16(tacc + c * 16, acc);
        const int at = t.begin + c * Sh::CHUNK + lane;
        int slot = -1;
        if (lane < Sh::CHUNK && at < t.end) {
          slot = __ldg(p.order + at);
          if (slot < 0 || slot >= p.S) slot = -1;
        }
        tmem_wait_ld();
        if (c + GROUPS >= chunks) {  // the last chunk is in registers: the accumulator goes back
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive_cluster(cluster_addr(&acc_empty[a], 0));
          released = true;
        }
        if constexpr (GLU) {
          // Gate warps finish columns 0 - 7 of the chunk, up warps 8 - 15; each hands the other its sums.
          float* mine = swap + ew * 256;
          const float* theirs = swap + partner * 256;
#pragma unroll
          for (int i = 0; i < 8; ++i)
            mine[i * 32 + lane] = __uint_as_float(up ? acc[i] : acc[8 + i]) + bias;
          asm volatile("bar.sync %0, 64;" ::"r"(bar) : "memory");
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const float here = __uint_as_float(up ? acc[8 + i] : acc[i]) + bias, there = theirs[i * 32 + lane];
            const float gate = up ? there : here, lin = up ? here : there;
            const int s = __shfl_sync(0xffffffffu, slot, (up ? 8 : 0) + i);
            if (nv && s >= 0) out[s * p.ldy] = Val<OT>::to(gate / (1.0f + expf(-gate)) * lin);
          }
          asm volatile("bar.sync %0, 64;" ::"r"(bar) : "memory");  // read before the next chunk's are written
        } else {
#pragma unroll
          for (int i = 0; i < Sh::CHUNK; ++i) {
            const int s = __shfl_sync(0xffffffffu, slot, i);
            if (nv && s >= 0) out[s * p.ldy] = Val<OT>::to(__uint_as_float(acc[i]) + bias);
          }
        }
      }
      if (!released) {
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive_cluster(cluster_addr(&acc_empty[a], 0));
      }
    }
    // Slots of no group: rows of zeros.
    const int none = group_begin(p.offsets, p.E, p.S);
    for (int64_t i = none + static_cast<int64_t>(blockIdx.x) * Sh::EPI + ew; i < p.S;
         i += static_cast<int64_t>(gridDim.x) * Sh::EPI) {
      const int s = __ldg(p.order + i);
      if (s < 0 || s >= p.S) continue;
      OV* out = static_cast<OV*>(p.y) + s * p.ldy;
      for (int64_t j = lane; j < p.n; j += 32) out[j] = Val<OT>::to(0.0f);
    }
  } else if (warp < 2 + Sh::EPI + Sh::CONV) {
    // -------------------------------------------- Q4_0: nibbles to the A tile
    if constexpr (Q4) {
      // Groups of four warps take turns at the stages: while one group's stage is on its way to the tensor core the
      // other widens the next.  A thread has a row of the CTA's 128, and its two blocks of the stage.
      const int ct = threadIdx.x - (2 + Sh::EPI) * 32;
      const int r = ct & 127, turn = ct >> 7;
      const uint32_t full0 = cluster_addr(a_full, 0);
      uint32_t stage = 0, phase = 0, raw = 0, raw_phase = 0, n = 0;
      bool ok = true;
      for (int tile = cluster; ok && tile < num_tiles; tile += nclusters) {
        const IdTile t = id_tile<GLU>(p, pre, tile, w_tiles, rank);
        const int64_t first = static_cast<int64_t>(t.e) * p.rows + (r < 64 ? t.r0 : t.r1);
        const int scale_at = 2 * kRawBox + (r >> 6) * kScaleBox + (static_cast<int>(first & 7) + (r & 63)) * 2;
        for (int ks = 0; ks < kst; ++ks, ++n) {
          if (ks % 4 == 0)
            ok = __all_sync(0xffffffffu, mbar_wait(&raw_full[raw], raw_phase, status, kDevWaitProducer, abort_flag));
          if (!ok) break;
          const bool mine = n % (Sh::CONV / 4) == static_cast<uint32_t>(turn);
          uint4 q[2];
          uint32_t d[2];
          if (mine) {
            const uint8_t* rb = raws + raw * kRawStride;
#pragma unroll
            for (int b = 0; b < 2; ++b) {
              const int block = (ks % 4) * 2 + b;
              q[b] = *reinterpret_cast<const uint4*>(rb + r * 128 + ((block ^ (r & 7)) << 4));
              d[b] = *reinterpret_cast<const uint16_t*>(rb + scale_at + block * (kScaleCols * 2));
            }
          }
          if (ks % 4 == 3 || ks == kst - 1) {
            __syncwarp();
            if (lane == 0) mbar_arrive(&raw_empty[raw]);
            if (++raw == RS) {
              raw = 0;
              raw_phase ^= 1u;
            }
          }
          if (mine) {
            ok = __all_sync(0xffffffffu, mbar_wait(&a_empty[stage], phase ^ 1u, status, kDevWaitProducer, abort_flag));
            if (!ok) break;
            uint8_t* ab = smem + stage * Sh::A + r * 128;
            constexpr uint32_t m = 0x0f0f0f0fu;
#pragma unroll
            for (int b = 0; b < 2; ++b) {
              // d as a number of 7 bits and one of 4: both times q - 8 are exact in fp16
              const uint32_t d2 = d[b] | (d[b] << 16), hi2 = d2 & 0xfff0fff0u, lo2 = hsub2_u(d2, hi2);
              const uint32_t words[4] = {q[b].x, q[b].y, q[b].z, q[b].w};
#pragma unroll
              for (int j = 0; j < 4; ++j) {  // values 8 j .. 8 j + 7: low nibbles of 8 bytes, then the high ones
                const uint32_t w0 = words[(j & 1) * 2], w1 = words[(j & 1) * 2 + 1];
                const uint2 u = codes4((j < 2 ? w0 : w0 >> 4) & m), v = codes4((j < 2 ? w1 : w1 >> 4) & m);
                uint4* at = reinterpret_cast<uint4*>(ab + (((b * 4 + j) ^ (r & 7)) << 4));
                at[0] = make_uint4(hmul2_u(u.x, hi2), hmul2_u(u.y, hi2), hmul2_u(v.x, hi2), hmul2_u(v.y, hi2));
                at[kABytes / 16] = make_uint4(hmul2_u(u.x, lo2), hmul2_u(u.y, lo2), hmul2_u(v.x, lo2), hmul2_u(v.y, lo2));
              }
            }
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive_remote(full0 + stage * 8);
          }
          if (++stage == AS) {
            stage = 0;
            phase ^= 1u;
          }
        }
      }
    }
  } else if (warp < 2 + Sh::EPI + Sh::CONV + Sh::GATHER) {
    // -------------------------------------------------------- rows of x by their numbers
    const int gw = warp - (2 + Sh::EPI + Sh::CONV);
    const int chunk = lane & 7;  // 16 bytes of a row's 128; four rows a request of the warp
    const int row0 = gw * 4 + (lane >> 3);
    uint32_t stage = 0, phase = 0;
    bool ok = true;
    for (int tile = cluster; ok && tile < num_tiles; tile += nclusters) {
      const IdTile t = id_tile<GLU>(p, pre, tile, w_tiles, rank);
      const int half = t.width >> 1;
      const uint8_t* src[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {  // the numbers behind the tile's last slot bring some row that exists; nobody looks at it
        const int s = __ldg(p.order + max(0, min(t.begin + static_cast<int>(rank) * half + i * 16 + row0, t.end - 1)));
        src[i] = static_cast<const uint8_t*>(p.x) + (s < 0 || s >= p.S ? 0 : s / p.per_row) * p.ldx * 2 + chunk * 16;
      }
      for (int ks = 0; ks < kst; ++ks) {
        ok = __all_sync(0xffffffffu, mbar_wait(&b_empty[stage], phase ^ 1u, status, kDevWaitProducer, abort_flag));
        if (!ok) break;
        const uint32_t dst = smem_u32(smem + Sh::OFF_B + stage * kBBytes) + ((chunk ^ (row0 & 7)) << 4) + row0 * 128;
        const int bytes = ks * kStageK + chunk * 8 < p.K ? 16 : 0;  // zeros behind the row's end
        const int64_t at = bytes ? static_cast<int64_t>(ks) * 128 : 0;
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (i * 16 < half)
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst + i * 2048), "l"(src[i] + at), "r"(bytes)
                         : "memory");
        asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(&x_full[stage])) : "memory");
        if (++stage == BS) {
          stage = 0;
          phase ^= 1u;
        }
      }
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
  } else {
    // A thread with no copies of its own makes the arrived rows visible to the tensor core (the same fence in a
    // gather warp would wait for all that the warp has asked for) and reports them to the leader.
    if (elect_one()) {
      const uint32_t full0 = cluster_addr(b_full, 0);
      uint32_t stage = 0, phase = 0;
      bool ok = true;
      for (int tile = cluster; ok && tile < num_tiles; tile += nclusters)
        for (int ks = 0; ks < kst; ++ks) {
          ok = mbar_wait(&x_full[stage], phase, status, kDevWaitProducer, abort_flag);
          if (!ok) break;
          fence_proxy_async_smem();
          mbar_arrive_remote(full0 + stage * 8);
          if (++stage == BS) {
            stage = 0;
            phase ^= 1u;
          }
        }
    }
  }

  tc_fence_before();
  __syncthreads();
  cluster_sync();  // the leader's MMAs into this CTA's TMEM and its reads of this CTA's stages are over
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc_pair(tmem_base, kAccs * kBN);
  }
}

template <int W, bool GLU, bool OUT32>
cudaError_t launch_shape(const MulMatIdArgs& a, const IdMaps& maps, int64_t tiles, cudaStream_t s) {
  using Sh = IdShape<W, GLU>;
  auto kernel = mul_mat_id_kernel<W, GLU, OUT32>;
  // Once per device: the shared memory, and how many pairs can be resident at once.
  static std::atomic<uint64_t> ready{0};
  static std::atomic<int> max_clusters[64];
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return cudaErrorInvalidDevice;
  const uint64_t bit = uint64_t{1} << dev;
  if (!(ready.load(std::memory_order_acquire) & bit)) {
    if (cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, Sh::SMEM)) return e;
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = 2;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.gridDim = dim3(2);
    cfg.blockDim = dim3(Sh::THREADS);
    cfg.dynamicSmemBytes = Sh::SMEM;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    int n = 0;
    if (cudaError_t e = cudaOccupancyMaxActiveClusters(&n, kernel, &cfg)) return e;
    if (n < 1) return cudaErrorInvalidConfiguration;
    max_clusters[dev].store(n);
    ready.fetch_or(bit, std::memory_order_acq_rel);
  }
  const unsigned pairs = static_cast<unsigned>(std::min<int64_t>(tiles, max_clusters[dev].load()));
  return launch_early(kernel, dim3(2 * pairs), dim3(Sh::THREADS), Sh::SMEM, s, 2, maps, a);
}

}  // namespace

cudaError_t launch_mul_mat_id(const MulMatIdArgs& a, int wtype, int xtype, int ytype, int num_sms, cudaStream_t s) {
  if (wtype == kWQ4 && a.S <= kFewRows * a.E && id_rows_fits(a.K)) return launch_id_rows(a, ytype, num_sms, s);
  const bool q4 = wtype == kWQ4, glu = a.glu != 0, out32 = ytype == kXF32;
  const CUtensorMapDataType dt = xtype == kXBF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  IdMaps maps = {};
  bool ok;
  if (q4) {
    ok = make_tensor_map_2d(&maps.w, CU_TENSOR_MAP_DATA_TYPE_UINT8, a.w, a.K / 2, a.E * a.rows, a.K / 2, kRawK / 2, 64,
                                  CU_TENSOR_MAP_SWIZZLE_128B) &&
         make_tensor_map_2d(&maps.scales, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, a.scales, a.lds, a.K / 32, a.lds * 2,
                            kScaleCols, kRawK / 32, CU_TENSOR_MAP_SWIZZLE_NONE);
  } else {
    // [expert][gate / up][row][k]: one box has a CTA's rows, with GLU 64 of either half
    const uint64_t dims[4] = {static_cast<uint64_t>(a.K), static_cast<uint64_t>(a.n), glu ? 2u : 1u,
                              static_cast<uint64_t>(a.E)};
    const uint64_t strides[3] = {static_cast<uint64_t>(a.ldw) * 2, static_cast<uint64_t>(a.ldw * a.n) * 2,
                                 static_cast<uint64_t>(a.E > 1 ? a.expert_stride : a.ldw * a.rows) * 2};
    const uint32_t box[4] = {kStageK, static_cast<uint32_t>(glu ? kBM / 2 : kBM), glu ? 2u : 1u, 1};
    ok = make_tensor_map_4d(&maps.w, dt, a.w, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B);
  }
  if (!ok) return cudaErrorInvalidValue;
  // As many tiles as there can be at most, whatever the groups' sizes.
  const int64_t w_tiles = (a.n + (glu ? kBM : 2 * kBM) - 1) / (glu ? kBM : 2 * kBM);
  const int64_t tiles = w_tiles * (a.S / kBN + std::min<int64_t>(a.E, a.S));
  if (tiles > INT32_MAX) return cudaErrorInvalidValue;
  auto pick = [&](auto w) {
    constexpr int W = decltype(w)::value;
    return glu ? (out32 ? launch_shape<W, true, true>(a, maps, tiles, s) : launch_shape<W, true, false>(a, maps, tiles, s))
               : (out32 ? launch_shape<W, false, true>(a, maps, tiles, s) : launch_shape<W, false, false>(a, maps, tiles, s));
  };
  if (q4) return pick(std::integral_constant<int, kWQ4>());
  return wtype == kXBF16 ? pick(std::integral_constant<int, kXBF16>()) : pick(std::integral_constant<int, kXF16>());
}

cudaError_t read_id_status(unsigned int* value, bool clear) {
  cudaError_t e = cudaMemcpyFromSymbol(value, g_id_status, sizeof(unsigned int));
  if (e != cudaSuccess || !clear) return e;
  const unsigned int zero = 0;
  return cudaMemcpyToSymbol(g_id_status, &zero, sizeof(unsigned int));
}

}  // namespace b2q
