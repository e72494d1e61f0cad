// The bf16 products outside the NVFP4 layers (a linear layer with its epilogue, the head with its loss): parameters and epilogue
// arithmetic that the kernels of dense_gemm.cu and dense_small.cu share.
#pragma once

#include "gemm_common.cuh"

#include <cuda_fp16.h>

#include <atomic>
#include <utility>

namespace metis {

struct DenseParams {
  int64_t M, N, K;
  int32_t* status;
  int32_t band;                                            // row tiles per band of the tile order
  // linear layer: d = act(z) * gate + residual with z = A B^T + bias; for the gradients act(z) in bf16 and act'(z) as half_slopes has it
  const void* bias;  int32_t bias_f32;
  int32_t act;
  const __nv_bfloat16* gate;      int64_t ldgate;  int32_t gate_wide;       // *_wide: rows of 16-byte pieces
  const __nv_bfloat16* residual;  int64_t ldr;     int32_t residual_wide;
  __nv_bfloat16* d;               int64_t ldd;     int32_t d_wide;
  __nv_bfloat16* act_out;         int64_t ldact;                            // (both of 16-byte rows)
  uint32_t* slope;                int64_t ldslope;                          // (in elements of 16 bits)
  // head: logits l = scale * (A B^T); columns of the vocabulary [0, N) of this launch are [col0, col0 + N) of all
  const int64_t* target;  int64_t ignore;
  const int32_t* row_of;                                   // the rows that are not ignored, one after the other (null: all rows, as they lie)
  const int32_t* live;  int32_t live_is_k;                 // their number, in place of M, or of K where the rows are contracted (null: neither)
  int64_t stats_ld;
  int64_t vocab;  int64_t col0;
  float scale, scale_log2e;                                // 1 / temperature, and that times log2(e)
  float weight_scale;                                      // scale, with the sign of the loss
  float2* stats;                                           // [slots, stats_ld]: maximum of l log2(e) and sum of 2^(l log2(e) - maximum), the target's l left out
  float* stats_e;                                          // [slots, stats_ld]: sum of 2^(..) (l log2(e) - maximum), or null
  const float* lse;                                        // [M]
  const float* target_logp;                                // [M]: the target's log-probability
  const float* gout;  int32_t gout_stride;                 // gradient of each row's loss (stride 1), or of all, times *inv_count (null: 1)
  const float* inv_count;
  int32_t half, half_rows;                                 // rows in two parts of bf16, so far apart (0: one part), and how many of each are rows
  // sum of pieces: fp32 addend.  With `splits` > 1 each split of the contraction has sums of its own, [splits, split_rows, N]
  const float* c;  int64_t ldc;
  int32_t splits, iters_per_split;
  int64_t split_rows;
};

extern std::atomic<int64_t> dense_launches;                // kernels launched by the entry points of these two files

// Lets a kernel take `bytes` of shared memory, asked once for each device (`done`: a bit for each that has it).
static inline cudaError_t allow_shared(const void* kernel, int bytes, std::atomic<uint64_t>& done) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  const uint64_t bit = dev < 64 ? (uint64_t)1 << dev : 0;
  if (done.load(std::memory_order_acquire) & bit) return cudaSuccess;
  e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e == cudaSuccess) done.fetch_or(bit, std::memory_order_release);
  return e;
}

// Products of few tokens (dense_small.cu).
struct SmallShape {
  int32_t rows;                                            // weight rows of a tile
  int32_t bn;                                              // tokens of a tile, a multiple of 16
  int32_t kb;                                              // blocks of 64 along the contraction to a stage
  int32_t stages, stage_bytes;
  int32_t splits, blocks_per_split;
};
struct SmallPlan {
  SmallShape sh;
  float us;
};
SmallPlan plan_dense_small(int64_t M, int64_t N, int64_t K, bool w_mn);
int32_t launch_dense_small(const SmallShape& sh, const void* t, int64_t ldt, const void* w, bool w_mn, int64_t ldw, const DenseParams& p, cudaStream_t st);
int32_t launch_dense_small_stats(const void* h, int64_t ldh, const void* w, int64_t ldw, const DenseParams& p, cudaStream_t st);
int64_t small_stats_slots(int64_t V);

#ifdef __CUDACC__

template <typename... KArgs, typename... Args>
static inline cudaError_t launch_counted(int launch_class, void (*kernel)(KArgs...), dim3 grid, dim3 block, size_t smem, cudaStream_t stream, Args&&... args) {
  dense_launches.fetch_add(1, std::memory_order_relaxed);
  return launch_overlapped(launch_class, kernel, grid, block, smem, stream, std::forward<Args>(args)...);
}

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

// A count that the kernel before wrote, read behind grid_dependency_wait().  Through a const __restrict__ pointer, or by __ldg, the compiler may
// take a load for one of memory that nobody writes and move it in front of that wait.
__device__ __forceinline__ int32_t load_count(const int32_t* p) {
  int32_t n;
  asm volatile("ld.global.b32 %0, [%1];" : "=r"(n) : "l"(p) : "memory");
  return n;
}

__device__ __forceinline__ float common_weight(const float* gout, const float* inv_count, float scale) { return *gout * (inv_count ? *inv_count : 1.0f) * scale; }

__device__ __forceinline__ float exp2_fast(float v) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}

// The logistic function 1 / (1 + exp(-u)); 0 where the exponential overflows.
__device__ __forceinline__ float logistic(float u) { return rcp_approx(1.0f + exp2_fast(-kLog2e * u)); }

// The normal distribution's function.  For a = |z| it is exp(-a^2 / 2) g(a) on the left, where g(a) = exp(a^2 / 2) erfc(a / sqrt 2) / 2
// falls like 1 / a: a polynomial in t = 1 / (1 + 0.3 a) without a constant term, fitted for least relative error over a in [0, 13.5] (where
// the value leaves fp32): 1.6e-7 by itself, 7e-7 in fp32 up to a = 3 and 8e-6 at the end, where a^2 is rounded.  16 instructions against the
// 40 of normcdff, which kept the tensor core waiting: 8192 x 8960 x 1536 with gelu 505 us.
__device__ __forceinline__ float normal_cdf(float z) {
  const float a = fabsf(z), t = rcp_approx(fmaf(0.3f, a, 1.0f));
  float g = fmaf(0.03593230992555618f, t, -0.1582782119512558f);
  g = fmaf(g, t, 0.20821012556552887f);
  g = fmaf(g, t, -0.05539681762456894f);
  g = fmaf(g, t, 0.12947063148021698f);
  g = fmaf(g, t, 0.09963709861040115f);
  g = fmaf(g, t, 0.12079841643571854f);
  g = fmaf(g, t, 0.11962638795375824f);
  const float left = g * t * exp2_fast(-0.7213475204444817f * a * a);
  return z < 0.0f ? left : 1.0f - left;
}

// act(z).  The forms keep their relative accuracy for large negative z (no difference of nearly equal numbers): silu and the tanh
// form of gelu are z times a logistic function, since (1 + tanh u) / 2 = 1 / (1 + exp(-2u)); the erf form is z times the
// normal distribution's function.
template <int kAct> __device__ __forceinline__ float activate(float z) {
  if constexpr (kAct == METIS_ACT_SILU) return z * logistic(z);
  if constexpr (kAct == METIS_ACT_GELU) return z * normal_cdf(z);
  if constexpr (kAct == METIS_ACT_GELU_TANH) return z * logistic(1.5957691216057308f * fmaf(0.044715f * z * z, z, z));      // u = 2 sqrt(2 / pi) (z + 0.044715 z^3)
  return z;
}
// act(z) and act'(z)
template <int kAct> __device__ __forceinline__ void activate_both(float z, float& a, float& slope) {
  a = z;
  slope = 1.0f;
  if constexpr (kAct == METIS_ACT_SILU) {
    const float p = logistic(z);
    a = z * p;
    slope = fmaf(a, 1.0f - p, p);
  }
  if constexpr (kAct == METIS_ACT_GELU) {
    const float p = normal_cdf(z);
    a = z * p;
    slope = fmaf(0.3989422804014327f * z, exp2_fast(-0.7213475204444817f * z * z), p);
  }
  if constexpr (kAct == METIS_ACT_GELU_TANH) {
    const float p = logistic(1.5957691216057308f * fmaf(0.044715f * z * z, z, z));
    a = z * p;
    slope = fmaf(a * (1.0f - p), 1.5957691216057308f * fmaf(0.134145f * z, z, 1.0f), p);
  }
}
// What a backward pass needs of z.  act' lies in [-0.13, 1.13], so 16 bits with ten of mantissa hold it: in fp16, times 2^15 (the values lie
// below 37100, and down to 2^-29 none loses bits).  An error of 2^-11 of the slope at most, an eighth of bf16's; from z in bf16 the slope has one of |z act''| 2^-9, and the
// gradients of x and W, which round dz to bf16, are then 1.7 times as far from the exact ones as their own last rounding puts them; 1.4 so.
constexpr float kSlopeScale = 32768.0f;
__device__ __forceinline__ uint32_t half_slopes(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo * kSlopeScale, hi * kSlopeScale);
  return *reinterpret_cast<const uint32_t*>(&h);
}
template <int kAct, int kN> __device__ __forceinline__ void activate_both_of(float (&v)[kN], uint32_t (&slopes)[kN / 2]) {
#pragma unroll
  for (int i = 0; i < kN / 2; ++i) {
    float s[2];
    activate_both<kAct>(v[2 * i], v[2 * i], s[0]);
    activate_both<kAct>(v[2 * i + 1], v[2 * i + 1], s[1]);
    slopes[i] = half_slopes(s[0], s[1]);
  }
}
template <int kN> __device__ __forceinline__ void activate_both_all(int act, float (&v)[kN], uint32_t (&slopes)[kN / 2]) {
  if (act == METIS_ACT_SILU) activate_both_of<METIS_ACT_SILU>(v, slopes);
  else if (act == METIS_ACT_GELU) activate_both_of<METIS_ACT_GELU>(v, slopes);
  else activate_both_of<METIS_ACT_GELU_TANH>(v, slopes);
}
template <int kN> __device__ __forceinline__ void activate_all(int act, float (&v)[kN]) {
  if (act == METIS_ACT_SILU) {
#pragma unroll
    for (int i = 0; i < kN; ++i) v[i] = activate<METIS_ACT_SILU>(v[i]);
  } else if (act == METIS_ACT_GELU) {
#pragma unroll
    for (int i = 0; i < kN; ++i) v[i] = activate<METIS_ACT_GELU>(v[i]);
  } else if (act == METIS_ACT_GELU_TANH) {
#pragma unroll
    for (int i = 0; i < kN; ++i) v[i] = activate<METIS_ACT_GELU_TANH>(v[i]);
  }
}

__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  const __nv_bfloat162 w = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&w);
}

__device__ __forceinline__ uint4 pack8(const float (&v)[8]) { return make_uint4(pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3]), pack_bf16(v[4], v[5]), pack_bf16(v[6], v[7])); }

// Running softmax statistics of one row: m, the maximum of the logits seen (times log2 e), s, the sum of 2^(l - m), and e, the
// sum of 2^(l - m) (l - m).  m starts at -infinity; base() replaces it there, so that no difference of two infinities is formed.
struct RowStats {
  float m, s, e;
};
constexpr uint32_t kMinusInfinity = 0xff800000u;         // (a logit that adds nothing)
__device__ __forceinline__ float stats_base(float m) { return m == -INFINITY ? 0.0f : m; }
// b into a
template <bool kEntropy> __device__ __forceinline__ void stats_merge(RowStats& a, const RowStats& b) {
  const float m = fmaxf(a.m, b.m), base = stats_base(m);
  const float fa = exp2_fast(a.m - base), fb = exp2_fast(b.m - base);
  if constexpr (kEntropy) {
    // (an empty side has e = 0; its distance is -infinity)
    const float da = a.m == -INFINITY ? 0.0f : a.m - base, db = b.m == -INFINITY ? 0.0f : b.m - base;
    a.e = fmaf(fa, fmaf(da, a.s, a.e), fb * fmaf(db, b.s, b.e));
  }
  a.s = fmaf(a.s, fa, b.s * fb);
  a.m = m;
}

#endif  // __CUDACC__

}  // namespace metis
