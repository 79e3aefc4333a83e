// b2q_groups.cuh -- what the kernels share whose rows are sorted by group (an
// expert, an adapter): 16-bit values, and the tile of a group that a CTA works on.
#pragma once

#include <atomic>
#include <cstdint>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <utility>

namespace b2q {

// Lets a kernel have more than 48 KB of dynamic shared memory; once per device.
template <auto KERNEL>
cudaError_t allow_smem(int bytes) {
  static std::atomic<uint64_t> done{0};
  int dev = 0;
  if (cudaError_t e = cudaGetDevice(&dev)) return e;
  const uint64_t bit = dev < 64 ? uint64_t{1} << dev : 0;
  if (done.load(std::memory_order_acquire) & bit) return cudaSuccess;
  if (cudaError_t e = cudaFuncSetAttribute(KERNEL, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes)) return e;
  done.fetch_or(bit, std::memory_order_acq_rel);
  return cudaSuccess;
}

// A launch that may begin while the stream's last kernel ends: its blocks are set
// up and then wait (grid_wait) for that kernel to be over and its writes to be
// seen.  Nothing of global memory is read or written before grid_wait.
// Measured: 1 to 2 us less per call where calls follow one another.
__device__ __forceinline__ void grid_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
template <typename... P, typename... A>
cudaError_t launch_early(void (*kernel)(P...), dim3 grid, dim3 block, size_t smem, cudaStream_t s, int cluster, A&&... args) {
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = static_cast<unsigned>(cluster);
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cfg.attrs = attr;
  cfg.numAttrs = cluster > 1 ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, kernel, std::forward<A>(args)...);
}

// 16 bytes into shared memory, zeros where there is nothing.  (256 bytes of a row come into the L2 at once: its next
// pieces are asked for soon.)
__device__ __forceinline__ void cp16(uint32_t dst, const void* src, bool there) {
  asm volatile("cp.async.cg.shared.global.L2::256B [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(there ? 16 : 0) : "memory");
}

// Values of type kXF32 / kXF16 / kXBF16 as fp32, and back with one rounding.
template <int T>
struct Val;
template <>
struct Val<0> {
  using type = float;
  static __device__ __forceinline__ float load(const float* p) { return *p; }
  static __device__ __forceinline__ float to(float v) { return v; }
};
template <>
struct Val<1> {
  using type = __half;
  static __device__ __forceinline__ float load(const __half* p) { return __half2float(*p); }
  static __device__ __forceinline__ __half to(float v) { return __float2half_rn(v); }
};
template <>
struct Val<2> {
  using type = __nv_bfloat16;
  static __device__ __forceinline__ float load(const __nv_bfloat16* p) { return __bfloat162float(*p); }
  static __device__ __forceinline__ __nv_bfloat16 to(float v) { return __float2bfloat16_rn(v); }
};

// N values (1, or as many as 4 or 8) in one load or store of their size; Raw: as
// they are loaded, which takes half the registers for 16-bit values.
template <int T, int N>
struct Raw {
  uint32_t w[T == 0 ? N : N / 2];
};
template <int T>
struct Raw<T, 1> {
  typename Val<T>::type v;
};
template <int T, int N>
__device__ __forceinline__ Raw<T, N> load_raw(const typename Val<T>::type* p) {
  Raw<T, N> r;
  if constexpr (N == 1) {
    r.v = *p;
  } else {
    constexpr int WORDS = T == 0 ? N : N / 2;
    if constexpr (WORDS == 2) {
      const uint2 u = *reinterpret_cast<const uint2*>(p);
      r.w[0] = u.x, r.w[1] = u.y;
    } else {
#pragma unroll
      for (int i = 0; i < WORDS; i += 4) {
        const uint4 u = *reinterpret_cast<const uint4*>(reinterpret_cast<const uint32_t*>(p) + i);
        r.w[i] = u.x, r.w[i + 1] = u.y, r.w[i + 2] = u.z, r.w[i + 3] = u.w;
      }
    }
  }
  return r;
}
template <int T, int N>
__device__ __forceinline__ void from_raw(const Raw<T, N>& r, float (&v)[N]) {
  if constexpr (N == 1) {
    v[0] = Val<T>::load(&r.v);
  } else if constexpr (T == 0) {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = __uint_as_float(r.w[i]);
  } else {
#pragma unroll
    for (int i = 0; i < N / 2; ++i) {
      if constexpr (T == 1) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&r.w[i]));
        v[2 * i] = f.x, v[2 * i + 1] = f.y;
      } else {
        v[2 * i] = __uint_as_float(r.w[i] << 16), v[2 * i + 1] = __uint_as_float(r.w[i] & 0xffff0000u);
      }
    }
  }
}
template <int T, int N>
__device__ __forceinline__ void load_vec(const typename Val<T>::type* p, float (&v)[N]) {
  from_raw<T, N>(load_raw<T, N>(p), v);
}
template <int T, int N>
__device__ __forceinline__ void store_vec(typename Val<T>::type* p, const float (&v)[N]) {
  if constexpr (N == 1) {
    *p = Val<T>::to(v[0]);
  } else if constexpr (T == 0) {
#pragma unroll
    for (int i = 0; i < N; i += 4) *reinterpret_cast<float4*>(p + i) = make_float4(v[i], v[i + 1], v[i + 2], v[i + 3]);
  } else {
    uint32_t w[N / 2];
#pragma unroll
    for (int i = 0; i < N / 2; ++i) {
      if constexpr (T == 1) {
        const __half2 h = __floats2half2_rn(v[2 * i], v[2 * i + 1]);
        w[i] = *reinterpret_cast<const uint32_t*>(&h);
      } else {
        const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
        w[i] = *reinterpret_cast<const uint32_t*>(&h);
      }
    }
    if constexpr (N == 8) *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
    else *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
  }
}

// The sorted slots of a group, from offsets that are not trusted: a stale or
// broken plan must not lead outside the S slots.  Group `groups` is the slots
// that have none, behind the last group's.
__device__ __forceinline__ int group_begin(const int32_t* offsets, int g, int64_t S) {
  return static_cast<int>(min(max(static_cast<int64_t>(__ldg(offsets + g)), int64_t{0}), S));
}
__device__ __forceinline__ int group_end(const int32_t* offsets, int g, int groups, int64_t S, int begin) {
  if (g >= groups) return static_cast<int>(S);
  return max(begin, group_begin(offsets, g + 1, S));
}

struct GroupTile {
  int group;  // -1: no such tile
  int begin, end;
};

// Tile number `tile` of all groups' tiles of at most `rows` sorted slots, group
// after group, the slots of no group last.  All lanes of a warp call it.
__device__ __forceinline__ GroupTile find_group_tile(const int32_t* offsets, int groups, int64_t S, int tile, int rows) {
  const int lane = threadIdx.x & 31;
  int before = 0;
  for (int g0 = 0; g0 <= groups; g0 += 32) {
    const int g = g0 + lane;
    int lo = 0, hi = 0;
    if (g <= groups) {
      lo = group_begin(offsets, g, S);
      hi = group_end(offsets, g, groups, S, lo);
    }
    const int n = (hi - lo + rows - 1) / rows;
    int inc = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int u = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += u;
    }
    const unsigned found = __ballot_sync(0xffffffffu, before + inc > tile);
    if (found) {
      const int src = __ffs(found) - 1;
      const int first = __shfl_sync(0xffffffffu, before + inc - n, src);
      GroupTile t;
      t.group = g0 + src;
      t.begin = __shfl_sync(0xffffffffu, lo, src) + (tile - first) * rows;
      t.end = min(t.begin + rows, __shfl_sync(0xffffffffu, hi, src));
      return t;
    }
    before += __shfl_sync(0xffffffffu, inc, 31);
  }
  return {-1, 0, 0};
}

}  // namespace b2q
