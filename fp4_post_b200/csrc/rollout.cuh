// What the kernels of a rollout share: indices of either width, the cache's addresses, sums over a block.
#pragma once

#include <atomic>

#include "common.cuh"

namespace metis {

void count_rollout_launches(int n);

// The cache as the kernels see it: metis_cache, checked.
struct CacheView {
  char* pool;
  int64_t page_bytes;       // of one page, all layers
  int64_t pages;
  int32_t* tables;
  int64_t sequences, width;
  int32_t* lengths;
  int32_t* refs;
  int32_t* status;
  int32_t* refused;         // [sequences], or null
  int32_t layers, kv_heads, page_size, head_dim, item;      // item: bytes of an element
};
int32_t check_cache(const metis_cache* c, CacheView* view);

#ifdef __CUDACC__

// Lets a kernel take `bytes` of shared memory, asked once for each device.
template <auto kKernel>
cudaError_t allow_smem(int bytes) {
  static std::atomic<uint64_t> done{0};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  const uint64_t bit = dev < 64 ? (uint64_t)1 << dev : 0;
  if (done.load(std::memory_order_acquire) & bit) return cudaSuccess;
  e = cudaFuncSetAttribute(kKernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e == cudaSuccess) done.fetch_or(bit, std::memory_order_release);
  return e;
}

__device__ __forceinline__ int64_t load_index(const void* p, bool wide, int64_t i) {
  return wide ? static_cast<const int64_t*>(p)[i] : (int64_t)static_cast<const int32_t*>(p)[i];
}

// Sums over the block of `kThreads` threads: what the threads before this one have, that with its own, and all.  Integers, or doubles in a
// fixed order; what one thread gets up to itself is bit for bit what the next one has before itself.  `warp_sums` has room for one value
// per warp; all threads call it.
// Of values that are not negative the sums never fall from one thread to the next, and do not move over one that adds nothing, whatever the roundings: a
// lane's is the whole lower half's sum plus its own within the upper half, half by half, and rounding keeps the order of sums with a common term.  (Where each lane adds the
// sum 1, 2, 4, ... lanes before it, neighbours' sums have other terms in common: one in a thousand borders between two of 512 tokens was a step of 64 bits above the next
// one, and a mark there was met by two threads, or by one that had no token.)
template <typename T> struct Scan { T before, upto, all; };
// The lane, read anew: of one that is known already the five conditions below are formed once and kept in a kernel's registers from scan to scan (sampling: 40 to 90 spilled words more,
// 6.8 us for 24 rows of 97 logits, 6.4 so).
__device__ __forceinline__ int lane_again() {
  int lane;
  asm volatile("mov.u32 %0, %%laneid;" : "=r"(lane));
  return lane;
}
template <typename T> __device__ __forceinline__ T lower_half(T v, int o) { return __shfl_sync(0xffffffffu, v, o - 1, 2 * o); }      // of 2 o lanes: its last lane's value
template <int kThreads, typename T>
__device__ __forceinline__ Scan<T> block_scan(T v, T* warp_sums) {
  constexpr int kWarps = kThreads / 32;
  const int lane = lane_again(), warp = threadIdx.x >> 5;
  T sum = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const T from = lower_half(sum, o);
    if (lane & o) sum += from;
  }
  __syncthreads();                                   // (warp_sums may still be read from the call before)
  if (lane == 31) warp_sums[warp] = sum;
  __syncthreads();
  T ahead = T(0), all = T(0);
#pragma unroll
  for (int w = 0; w < kWarps; ++w) {
    if (w == warp) ahead = all;
    all += warp_sums[w];
  }
  const T left = __shfl_up_sync(0xffffffffu, sum, 1);
  return {lane == 0 ? ahead : ahead + left, ahead + sum, all};
}
// Two at once, between the same barriers.
template <int kThreads, typename T>
__device__ __forceinline__ void block_scan_two(T a, T b, T* sums_a, T* sums_b, Scan<T>& of_a, Scan<T>& of_b) {
  constexpr int kWarps = kThreads / 32;
  const int lane = lane_again(), warp = threadIdx.x >> 5;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const T from_a = lower_half(a, o), from_b = lower_half(b, o);
    if (lane & o) { a += from_a; b += from_b; }
  }
  __syncthreads();
  if (lane == 31) { sums_a[warp] = a; sums_b[warp] = b; }
  __syncthreads();
  T ahead_a = T(0), ahead_b = T(0), all_a = T(0), all_b = T(0);
#pragma unroll
  for (int w = 0; w < kWarps; ++w) {
    if (w == warp) { ahead_a = all_a; ahead_b = all_b; }
    all_a += sums_a[w];
    all_b += sums_b[w];
  }
  const T left_a = __shfl_up_sync(0xffffffffu, a, 1), left_b = __shfl_up_sync(0xffffffffu, b, 1);
  of_a = {lane == 0 ? ahead_a : ahead_a + left_a, ahead_a + a, all_a};
  of_b = {lane == 0 ? ahead_b : ahead_b + left_b, ahead_b + b, all_b};
}
template <int kThreads, typename T>
__device__ __forceinline__ T block_exclusive(T v, T* warp_sums, T& total) {
  const Scan<T> s = block_scan<kThreads>(v, warp_sums);
  total = s.all;
  return s.before;
}

#endif

}  // namespace metis
