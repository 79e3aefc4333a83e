// b2q_kv_plan.cu -- the page plan of a paged key / value cache, built on the
// device from the requests' lengths: which free pages each request takes for
// its new tokens, the cache slot and position of every new token, and the
// per-request offsets and lengths that the attention reads.
//
//   had_b  = ceil(cached_b / ps)          pages the request owns
//   need_b = ceil((cached_b + new_b) / ps)
//   base_b = sum_{i<b} (need_i - had_i)   its first entry of the free list
//   table[b][j] = free[base_b + j - had_b]  for had_b <= j < need_b, -1 after
//   token t of request b at position p:  slot = table[b][p / ps] * ps + p % ps
//
// One launch: every CTA scans all the lengths itself (two block scans over at
// most kPlanMaxB values that the L2 serves), so no CTA waits for another; then
// the CTAs share out the table rows (one warp a row) and the tokens (four
// consecutive ones per thread, one search in the scanned offsets).  The work is
// 12 bytes a token and 4 a table entry, all written once; bound by its latency
// (the launch, two scans, one pass of writes): 5.3 us for 48 requests of one
// token, 11.5 us for 1000 requests of 750k tokens in all, where the bytes are 1.5 us.
#include "b2q_internal.h"

namespace b2q {

namespace {

constexpr int kPlanThreads = 512;

// Exclusive scan over the block of one int64 per thread; *total is the sum.
__device__ __forceinline__ int64_t block_scan(int64_t v, int64_t* warp_sums, int64_t* total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int64_t inc = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t u = __shfl_up_sync(0xffffffffu, inc, o);
    if (lane >= o) inc += u;
  }
  __syncthreads();  // the sums of an earlier call are no longer read
  if (lane == 31) warp_sums[warp] = inc;
  __syncthreads();
  int64_t before = 0, all = 0;
#pragma unroll
  for (int w = 0; w < kPlanThreads / 32; ++w) {
    const int64_t u = warp_sums[w];
    if (w < warp) before += u;
    all += u;
  }
  *total = all;
  return before + inc - v;
}

struct PlanArgs {
  const int32_t* cached;
  const int32_t* fresh;
  int B;
  int page_shift;
  const int32_t* free_pages;
  int64_t n_free;
  int32_t* table;
  int64_t width, ldt;
  int64_t max_tokens;
  int64_t* slots;
  int32_t* pos;
  int32_t* cu;
  int32_t* kv_len;
  int32_t* counts;
};

__device__ __forceinline__ int32_t sat32(int64_t v) { return v > INT32_MAX ? INT32_MAX : static_cast<int32_t>(v); }

__global__ void __launch_bounds__(kPlanThreads) kv_plan_kernel(const PlanArgs a) {
  extern __shared__ int32_t plan_smem[];
  __shared__ int64_t warp_sums[kPlanThreads / 32];
  int32_t* s_cu = plan_smem;               // [B + 1] first token of each request
  int32_t* s_base = plan_smem + a.B + 1;   // [B] first free-list entry of each request
  const int tid = threadIdx.x;
  const int64_t ps1 = (int64_t{1} << a.page_shift) - 1;

  int64_t tok0 = 0, page0 = 0, lost = 0;
  for (int b0 = 0; b0 < a.B; b0 += kPlanThreads) {
    const int b = b0 + tid;
    const int64_t c = b < a.B ? max(a.cached[b], 0) : 0;
    const int64_t n = b < a.B ? max(a.fresh[b], 0) : 0;
    int64_t total;
    const int64_t at = tok0 + block_scan(n, warp_sums, &total);
    tok0 += total;
    // tokens past max_tokens are not planned
    const int64_t lo = min(at, a.max_tokens), hi = min(at + n, a.max_tokens);
    const int64_t had = min((c + ps1) >> a.page_shift, a.width);
    const int64_t need = max(had, min((c + (hi - lo) + ps1) >> a.page_shift, a.width));
    const int64_t base = page0 + block_scan(b < a.B ? need - had : 0, warp_sums, &total);
    page0 += total;
    if (b < a.B) {
      s_cu[b] = static_cast<int32_t>(lo);
      s_base[b] = sat32(base);
      if (blockIdx.x == 0) {
        a.cu[b] = static_cast<int32_t>(lo);
        a.kv_len[b] = sat32(c + (hi - lo));
        // tokens without a slot: those in an owned page that the table lacks,
        // and those past the pages that the free list can give
        const int64_t end = c + (hi - lo), own = min(end, had << a.page_shift);
        if (c < own && a.table[b * a.ldt + had - 1] < 0) lost += own - c;
        const int64_t got = had + min(need - had, max(a.n_free - base, int64_t{0}));
        lost += max(int64_t{0}, end - max(c, got << a.page_shift));
      }
    }
  }
  if (tid == 0) s_cu[a.B] = static_cast<int32_t>(min(tok0, a.max_tokens));
  if (blockIdx.x == 0) {
    int64_t total;
    block_scan(lost, warp_sums, &total);
    if (tid == 0) {
      a.cu[a.B] = static_cast<int32_t>(min(tok0, a.max_tokens));
      a.counts[0] = sat32(page0);
      a.counts[1] = sat32(total);
    }
  }
  __syncthreads();
  const int n_tok = s_cu[a.B];

  // table rows: entries past the pages the request owned
  const int lane = tid & 31;
  const int64_t warps = static_cast<int64_t>(gridDim.x) * (kPlanThreads / 32);
  for (int64_t b = static_cast<int64_t>(blockIdx.x) * (kPlanThreads / 32) + (tid >> 5); b < a.B; b += warps) {
    const int64_t c = max(a.cached[b], 0);
    const int64_t had = min((c + ps1) >> a.page_shift, a.width);
    const int64_t need = max(had, min((c + (s_cu[b + 1] - s_cu[b]) + ps1) >> a.page_shift, a.width));
    for (int64_t j = had + lane; j < a.width; j += 32) {
      const int64_t f = s_base[b] + (j - had);
      a.table[b * a.ldt + j] = j < need && f < a.n_free ? a.free_pages[f] : -1;
    }
  }

  // tokens, four at a time
  const int64_t threads = static_cast<int64_t>(gridDim.x) * kPlanThreads;
  for (int64_t t4 = (static_cast<int64_t>(blockIdx.x) * kPlanThreads + tid) * 4; t4 < a.max_tokens; t4 += threads * 4) {
    int64_t slot[4] = {-1, -1, -1, -1};
    int32_t pos[4] = {-1, -1, -1, -1};
    if (t4 < n_tok) {
      int b = 0, hi = a.B - 1;  // the last request whose first token is at or before t4
      while (b < hi) {
        const int mid = (b + hi + 1) >> 1;
        if (s_cu[mid] <= t4)
          b = mid;
        else
          hi = mid - 1;
      }
      int64_t c = -1, had = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int64_t t = t4 + i;
        if (t >= n_tok) break;
        if (t >= s_cu[b + 1]) c = -1;
        while (t >= s_cu[b + 1]) ++b;  // t < n_tok = s_cu[B], so this ends at b < B
        if (c < 0) {
          c = max(a.cached[b], 0);
          had = min((c + ps1) >> a.page_shift, a.width);
        }
        const int64_t p = c + (t - s_cu[b]);
        const int64_t j = p >> a.page_shift;
        int32_t page = -1;
        if (j < had) {
          page = a.table[b * a.ldt + j];
        } else if (j < a.width) {
          const int64_t f = s_base[b] + (j - had);
          if (f < a.n_free) page = a.free_pages[f];
        }
        pos[i] = sat32(p);
        if (page >= 0) slot[i] = (static_cast<int64_t>(page) << a.page_shift) + (p & ps1);
      }
    }
    if (t4 + 4 <= a.max_tokens) {
      *reinterpret_cast<longlong2*>(a.slots + t4) = make_longlong2(slot[0], slot[1]);
      *reinterpret_cast<longlong2*>(a.slots + t4 + 2) = make_longlong2(slot[2], slot[3]);
      *reinterpret_cast<int4*>(a.pos + t4) = make_int4(pos[0], pos[1], pos[2], pos[3]);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (t4 + i < a.max_tokens) {
          a.slots[t4 + i] = slot[i];
          a.pos[t4 + i] = pos[i];
        }
    }
  }
}

}  // namespace

cudaError_t launch_kv_plan(const int32_t* cached, const int32_t* fresh, int64_t B, int page_shift,
                           const int32_t* free_pages, int64_t n_free, int32_t* table, int64_t width, int64_t ldt,
                           int64_t max_tokens, int64_t* slots, int32_t* pos, int32_t* cu, int32_t* kv_len,
                           int32_t* counts, int num_sms, cudaStream_t s) {
  const int smem = static_cast<int>((2 * B + 1) * 4);
  if (smem > 48 * 1024) {
    const cudaError_t e = cudaFuncSetAttribute(kv_plan_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                               static_cast<int>((2 * kPlanMaxB + 1) * 4));
    if (e != cudaSuccess) return e;
  }
  // CTAs by the larger of the two fills, one pass each; at most one per SM.
  const int64_t by_tokens = (max_tokens + kPlanThreads * 4 - 1) / (kPlanThreads * 4);
  const int64_t by_rows = (B + kPlanThreads / 32 - 1) / (kPlanThreads / 32);
  int64_t grid = by_tokens > by_rows ? by_tokens : by_rows;
  if (grid > num_sms) grid = num_sms;
  if (grid < 1) grid = 1;
  PlanArgs a{cached, fresh, static_cast<int>(B), page_shift, free_pages, n_free, table, width, ldt,
             max_tokens, slots, pos, cu, kv_len, counts};
  kv_plan_kernel<<<static_cast<unsigned>(grid), kPlanThreads, smem, s>>>(a);
  return cudaGetLastError();
}

}  // namespace b2q
