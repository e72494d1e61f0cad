// One token for each row of logits: temperature, top-k, top-p, min-p, then the token at which the kept weights pass u times their sum.
//
//   w_i = exp((x_i - max x) (1/T)) in fp32 (1 at the maximum);  order: larger x first, equal ones by index
//   top-k keeps the first k of the order; top-p the shortest front of those whose weights are at least p of theirs; min-p those with w >= min_p.
//   Each keeps a front of the order, so that what is kept is "x above a cut, and the first n of those that equal it".
//
// A cluster of up to eight blocks takes a row: it is read once from memory, 16 bytes at a time, and stays in shared memory in fp32 for all passes.  Nothing is
// sorted: a cut is found by histograms of 2048 bins, first of (max - x) / T in steps of 1/64, then of the bits of the logits in the bin where
// the cut lies until one value is left (one more level for bf16, two or three for fp32).
//
// Whether a token is in or out goes by sums over up to all the vocabulary, and an fp32 sum would move borders with the order of its terms.  Here the
// sums have 64 bits: a bin's weights lie within a factor of 2^(1/44), all 24 bits of each are multiples of one unit, and the bin adds them as
// whole numbers (two of at most 14 bits: 20000 of those fit 32 bits), exactly and in any order; bins, threads and blocks are added as doubles in
// a fixed order.  So a token does not depend on the schedule, and two programs that take the same weights find the same one.
#include "rollout.cuh"

#include <cooperative_groups.h>
#include <math_constants.h>

namespace cg = cooperative_groups;

namespace metis {
namespace {

constexpr int kThreads = 512;
constexpr int kBins = 2048;
constexpr int kMaxCluster = 8;
constexpr float kStep = 64.0f;                     // bins for a factor of e
constexpr int kLowBits = 13;

struct SampleParams {
  const void* logits;
  int64_t ld;
  int32_t vocab, each;                             // each: elements of a thread, odd (their reads then meet no bank twice)
  int32_t dtype;
  bool u_64;
  const void* u;
  double top_p;
  float temperature, min_p;
  int32_t top_k;
  const float *temperature_rows, *top_p_rows, *min_p_rows;
  const int32_t* top_k_rows;
  int64_t* token;
  float* logprob;
};

struct Found { double above, inside; int32_t bin; };      // weight before the bin where the target is met, and in it

struct Shared {
  double sums[kThreads / 32];
  int64_t counts[kThreads / 32];
  double gathered[2][kMaxCluster];
  Found found;
  uint32_t low, high;                              // keys in the bin, of this block
  float maxima[kThreads / 32];
  uint32_t* lows;                                  // the two histograms, [kBins] each
  uint32_t* highs;
};

// The same order as the numbers', as whole numbers; bf16 in 16 bits.
__device__ __forceinline__ uint32_t key_of(float x, int drop) {
  const uint32_t b = __float_as_uint(x);
  return ((b & 0x80000000u) ? ~b : b | 0x80000000u) >> drop;
}
__device__ __forceinline__ float value_of(uint32_t key, int drop) {
  const bool positive = (key << drop) >> 31;
  const uint32_t b = (key << drop) | (!positive && drop ? (1u << drop) - 1u : 0u);
  return __uint_as_float(positive ? b & 0x7fffffffu : ~b);
}

// The cluster's blocks on one row.
struct Row {
  cg::cluster_group cluster;
  Shared& sh;
  const float* x;                                  // this block's logits; -inf behind the last
  int blocks, rank, held;                          // held: elements of x
  float top, inverse;                              // the largest logit, 1/T
  int drop;
  int turn = 0;

  __device__ float weight(float v) const { return v == top ? 1.0f : expf(__fmul_rn(__fsub_rn(v, top), inverse)); }

  // One value of each block to all; two buffers in turn, so that one barrier does for both writing and reading.
  __device__ const double* gather(double v) {
    turn ^= 1;
    if (threadIdx.x < (unsigned)blocks) cluster.map_shared_rank(&sh, threadIdx.x)->gathered[turn][rank] = v;
    cluster.sync();
    return sh.gathered[turn];
  }
  // What the blocks before this one have, and all.
  __device__ double ahead(double v, double& all) {
    const double* g = gather(v);
    double before = 0.0;
    all = 0.0;
    for (int r = 0; r < blocks; ++r) {
      if (r == rank) before = all;
      all += g[r];
    }
    return before;
  }

  __device__ int bin_of(float v) const {
    const float d = __fmul_rn(__fmul_rn(__fsub_rn(top, v), inverse), kStep);
    return v == top ? 0 : d < (float)(kBins - 1) ? (int)d : kBins - 1;
  }
  // The unit of a bin's weights is 2^unit_of: two bits below the last one of the smallest.  (What lies in the last bin, at most 2^-46 of the largest, loses what it
  // has below 2^-72.)
  __device__ static int unit_of(int bin) { return bin == kBins - 1 ? -72 : (int)floorf(-(float)(bin + 1) * (1.44269504f / kStep)) - 2 - 24; }
  __device__ static uint32_t whole(float w, int unit) { return (uint32_t)(w * __uint_as_float((uint32_t)(127 - unit) << 23)); }

  __device__ void clear() {
    for (int i = threadIdx.x; i < kBins; i += kThreads) sh.lows[i] = sh.highs[i] = 0u;
    __syncthreads();
  }
  template <bool kMass> __device__ void add(int bin, float v, int unit) {
    if constexpr (kMass) {
      const uint32_t m = whole(weight(v), unit);
      atomicAdd(&sh.lows[bin], m & ((1u << kLowBits) - 1u));
      atomicAdd(&sh.highs[bin], m >> kLowBits);
    } else {
      atomicAdd(&sh.lows[bin], 1u);
    }
  }
  // Where the bins' sums, in order, reach the target; false if they do not.  units: the bins' unit, or their own where it is 1.
  template <bool kMass> __device__ bool reach(double target, int unit, Found& out) {
    __syncthreads();
    cluster.sync();
    const int slice = kBins / blocks, mine = slice > kThreads ? slice / kThreads : 1;
    double v[kBins / kThreads], sum = 0.0;
    for (int i = 0; i < mine; ++i) {
      const int local = threadIdx.x * mine + i;
      v[i] = 0.0;
      if (local >= slice) continue;
      const int bin = rank * slice + local;
      uint64_t low = 0, high = 0;
      for (int r = 0; r < blocks; ++r) {
        low += cluster.map_shared_rank(sh.lows, r)[bin];
        if (kMass) high += cluster.map_shared_rank(sh.highs, r)[bin];
      }
      const uint64_t m = low + (high << kLowBits);
      if (m) v[i] = kMass ? ldexp((double)m, unit == 1 ? unit_of(bin) : unit) : (double)m;
      sum += v[i];
    }
    const Scan<double> s = block_scan<kThreads>(sum, sh.sums);
    double all;
    const double base = ahead(s.all, all);
    if (all < target) return false;                // the same for all blocks
    const double before = base + s.before, upto = base + s.upto;
    if (before < target && target <= upto) {
      double above = before;
      int hit = -1;
      for (int i = 0; i < mine; ++i) {
        if (v[i] == 0.0) continue;
        if (hit >= 0) {
          above += v[hit];
        }
        hit = i;
        if (target <= above + v[i]) break;
      }
      const Found f = {above, v[hit], rank * slice + (int)threadIdx.x * mine + hit};
      for (int r = 0; r < blocks; ++r) cluster.map_shared_rank(&sh, r)->found = f;
    }
    cluster.sync();
    out = sh.found;
    return true;
  }

  // The cut of the elements above `floor`: `at` such that the weights (or the number) of those above it are below the target and with those that equal
  // it are not; what is above, and how many equal it.  False if all of them do not reach the target.
  template <bool kMass> __device__ bool cut(double target, float floor, float& at, double& above, double& ties) {
    clear();
    for (int i = threadIdx.x; i < held; i += kThreads)
      if (x[i] > floor) {
        const int bin = bin_of(x[i]);
        add<kMass>(bin, x[i], kMass ? unit_of(bin) : 0);
      }
    Found f;
    if (!reach<kMass>(target, 1, f)) return false;
    above = f.above;
    const int bin = f.bin, unit = unit_of(bin);
    // the bin's smallest and largest keys
    if (threadIdx.x == 0) { sh.low = 0xffffffffu; sh.high = 0u; }
    __syncthreads();
    uint32_t low = 0xffffffffu, high = 0u;
    for (int i = threadIdx.x; i < held; i += kThreads)
      if (x[i] > floor && bin_of(x[i]) == bin) {
        const uint32_t k = key_of(x[i], drop);
        low = min(low, k);
        high = max(high, k);
      }
    low = __reduce_min_sync(0xffffffffu, low);
    high = __reduce_max_sync(0xffffffffu, high);
    if ((threadIdx.x & 31) == 0) { atomicMin(&sh.low, low); atomicMax(&sh.high, high); }
    __syncthreads();
    const double* g = gather((double)sh.low);
    for (int r = 0; r < blocks; ++r) low = min(low, (uint32_t)g[r]);
    g = gather((double)sh.high);
    for (int r = 0; r < blocks; ++r) high = max(high, (uint32_t)g[r]);
    while (true) {
      const uint32_t span = high - low;
      const int shift = max(0, 21 - __clz(span));          // (span >> shift) < 2048
      clear();
      for (int i = threadIdx.x; i < held; i += kThreads)
        if (x[i] > floor && bin_of(x[i]) == bin) {
          const uint32_t k = key_of(x[i], drop);
          if (k >= low && k <= high) add<kMass>((int)((high - k) >> shift), x[i], unit);
        }
      // (a target that rounding puts in front of the bin's first element, or behind its last, is met by that one)
      Found next;
      if (!reach<kMass>(fmax(fmin(target - above, f.inside), 1e-300), unit, next)) return false;
      above += next.above;
      f.inside = next.inside;
      high -= (uint32_t)next.bin << shift;
      if (shift == 0) break;
      low = max(low, high - ((1u << shift) - 1u));
    }
    at = value_of(high, drop);
    ties = kMass ? rint(f.inside / ldexp((double)whole(weight(at), unit), unit)) : f.inside;
    return true;
  }
};

template <typename T>
__global__ void __launch_bounds__(kThreads) sample_kernel(const SampleParams p) {
  extern __shared__ __align__(16) float dynamic[];
  __shared__ Shared sh;
  const cg::cluster_group cluster = cg::this_cluster();
  const int blocks = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
  const int64_t row = blockIdx.x / blocks;
  const int held = p.each * kThreads, first = rank * held, here = max(0, min(held, p.vocab - first));
  float* x = dynamic + 2 * kBins;
  if (threadIdx.x == 0) {
    sh.lows = reinterpret_cast<uint32_t*>(dynamic);
    sh.highs = reinterpret_cast<uint32_t*>(dynamic) + kBins;
  }
  cluster.barrier_arrive();                        // (a block is written to by the others once all have begun)
  grid_dependency_wait();

  // ---- the row; NaN and what is behind it as -inf, -0 as 0 ----
  float top = -CUDART_INF_F;
  const T* from = static_cast<const T*>(p.logits) + row * p.ld + first;
  auto take = [&](float v) {
    v = v == v ? v + 0.0f : -CUDART_INF_F;
    top = fmaxf(top, v);
    return v;
  };
  constexpr int kWide = 16 / sizeof(T);
  int done = 0;
  if ((reinterpret_cast<uintptr_t>(from) & 15) == 0) {
    done = here / kWide * kWide;
#pragma unroll 4
    for (int i = threadIdx.x * kWide; i < done; i += kThreads * kWide) {
      const uint4 w = __ldcs(reinterpret_cast<const uint4*>(from + i));
      float4* to = reinterpret_cast<float4*>(x + i);
      if constexpr (sizeof(T) == 2) {
        to[0] = make_float4(take(bf16_lo(w.x)), take(bf16_hi(w.x)), take(bf16_lo(w.y)), take(bf16_hi(w.y)));
        to[1] = make_float4(take(bf16_lo(w.z)), take(bf16_hi(w.z)), take(bf16_lo(w.w)), take(bf16_hi(w.w)));
      } else {
        to[0] = make_float4(take(__uint_as_float(w.x)), take(__uint_as_float(w.y)), take(__uint_as_float(w.z)), take(__uint_as_float(w.w)));
      }
    }
  }
  for (int i = done + threadIdx.x; i < held; i += kThreads) x[i] = i < here ? take((float)from[i]) : -CUDART_INF_F;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  if ((threadIdx.x & 31) == 0) sh.maxima[threadIdx.x >> 5] = top;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kThreads / 32; ++w) top = fmaxf(top, sh.maxima[w]);

  cluster.barrier_wait();
  Row r{cluster, sh, x, blocks, rank, held, 0.0f, 0.0f, sizeof(T) == 2 ? 16 : 0};
  {
    const double* g = r.gather((double)top);
    for (int i = 0; i < blocks; ++i) top = fmaxf(top, (float)g[i]);
  }
  const float t = p.temperature_rows ? p.temperature_rows[row] : p.temperature, min_p = p.min_p_rows ? p.min_p_rows[row] : p.min_p;
  const double top_p = p.top_p_rows ? (double)p.top_p_rows[row] : p.top_p;
  int64_t k = p.top_k_rows ? p.top_k_rows[row] : p.top_k;
  const double u = p.u_64 ? static_cast<const double*>(p.u)[row] : (double)static_cast<const float*>(p.u)[row];
  const bool fine = (t == 0.0f || (t >= 0x1p-126f && t <= 3.4028235e38f)) && top_p >= 0.0 && min_p >= 0.0f && min_p <= 1.0f && k >= 0 && u >= 0.0 && u < 1.0 &&
                    top > -CUDART_INF_F;
  if (!fine) {                                     // (for all blocks of the cluster)
    if (rank == 0 && threadIdx.x == 0) {
      p.token[row] = -1;
      if (p.logprob) p.logprob[row] = CUDART_NAN_F;
    }
    cluster.sync();
    return;
  }
  const float heat = t == 0.0f ? 1.0f : t;
  if (t == 0.0f) k = 1;
  r.top = top;
  r.inverse = __fdiv_rn(1.0f, heat);

  // ---- all weights, for the log-probability and where nothing but a share of all is asked for ----
  const int mine = threadIdx.x * p.each;
  double all_weights = 0.0;
  if (p.logprob || (top_p < 1.0 && k == 0)) {
    double sum = 0.0;
    for (int i = mine; i < mine + p.each; ++i) sum += (double)r.weight(x[i]);
    const Scan<double> s = block_scan<kThreads>(sum, sh.sums);
    r.ahead(s.all, all_weights);
  }

  // ---- the cut: kept are those above `at` and the first `ties` that equal it ----
  float at = -CUDART_INF_F;
  double ties = 0.0;
  double above;
  if (k == 1) {
    at = top;
    ties = 1.0;
  } else if (k > 0 && k < p.vocab) {
    float c;
    double equal;
    if (r.cut<false>((double)k, -CUDART_INF_F, c, above, equal)) {       // (else there are not so many)
      at = c;
      ties = (double)k - above;
    }
  }
  if (top_p < 1.0 && k != 1) {
    double total = all_weights;
    if (k > 0) {
      double sum = 0.0;
      for (int i = mine; i < mine + p.each; ++i) if (x[i] > at) sum += (double)r.weight(x[i]);
      const Scan<double> s = block_scan<kThreads>(sum, sh.sums);
      r.ahead(s.all, total);
      above = total;
      if (at > -CUDART_INF_F) total += ties * (double)r.weight(at);
    }
    const double target = fmax(top_p * total, 1e-300);            // (the first one is always kept)
    float c;
    double equal, before = 0.0;
    double limit = ties;
    bool found = r.cut<true>(target, at, c, before, equal);
    if (found) {
      at = c;
      limit = equal;
    } else {
      before = above;                              // all that are above the cut of top-k, and some that equal it
      found = k > 0 && at > -CUDART_INF_F;
    }
    if (found) {
      // of those that equal the cut, as many as have less than the target in front of them
      const double w = (double)r.weight(at);
      double n = w > 0.0 ? fmax(1.0, ceil((target - before) / w)) : limit;
      while (n < limit && before + n * w < target) n += 1.0;
      while (n > 1.0 && before + (n - 1.0) * w >= target) n -= 1.0;
      ties = fmin(n, limit);
    }
  }

  // ---- which of the equal ones this thread's first is ----
  double rank_of = 0.0;
  if (at > -CUDART_INF_F) {
    int64_t equal = 0;
    for (int i = mine; i < mine + p.each; ++i) equal += x[i] == at;
    const Scan<int64_t> s = block_scan<kThreads>(equal, sh.counts);
    double none;
    rank_of = r.ahead((double)s.all, none) + (double)s.before;
  }
  // ---- the kept weights in order of their indices ----
  auto walk = [&](const auto& keep) {
    double nth = rank_of;
    for (int i = mine; i < mine + p.each; ++i) {
      const float v = x[i];
      if (v < at || v == -CUDART_INF_F) continue;
      if (v == at) {
        nth += 1.0;
        if (nth > ties) continue;
      }
      const float w = r.weight(v);
      if (w >= min_p && w > 0.0f && !keep(i, w)) break;
    }
  };
  double sum = 0.0;
  walk([&](int, float w) { sum += (double)w; return true; });
  const Scan<double> s = block_scan<kThreads>(sum, sh.sums);
  double total;
  const double base = r.ahead(s.all, total);
  double mark = u * total;
  if (mark >= total) mark = __longlong_as_double(__double_as_longlong(total) - 1);      // (rounded up: the last one)
  const double before = base + s.before;
  if (before <= mark && mark < base + s.upto) {
    double acc = before;
    int token = -1;
    walk([&](int i, float w) {
      acc += (double)w;
      token = i;
      return acc <= mark;
    });
    p.token[row] = first + token;
    if (p.logprob) p.logprob[row] = (float)((x[token] == top ? 0.0 : ((double)x[token] - (double)top) / (double)heat) - log(all_weights));
  }
  cluster.sync();                                  // nobody leaves while another block may read what it has
}

}  // namespace
}  // namespace metis

using namespace metis;

extern "C" int32_t metis_sample(const metis_sample_args* a) {
  if (!a || !a->logits || !a->u || !a->token) return fail(METIS_ERR_BAD_ARGUMENT, "null pointer");
  if (a->dtype != METIS_DTYPE_BF16 && a->dtype != METIS_DTYPE_F32) return fail(METIS_ERR_BAD_ARGUMENT, "logits must be bf16 or fp32");
  if (a->rows <= 0 || a->vocab <= 0 || (a->rows > 1 && a->ld < a->vocab)) return fail(METIS_ERR_BAD_SHAPE, "rows and vocab must be positive, rows of logits apart");
  if (a->vocab > METIS_SAMPLE_MAX_VOCAB) return fail(METIS_ERR_TOO_LARGE, "vocabularies have at most %d entries", METIS_SAMPLE_MAX_VOCAB);
  // A block for each 8192 entries up to eight of them: fewer entries for each are sooner done, more blocks wait longer for one another.
  int blocks = 1;
  while (blocks < kMaxCluster && a->vocab > (int64_t)blocks * 8192) blocks *= 2;
  int64_t each = ceil_div(ceil_div(a->vocab, blocks), kThreads);
  each |= 1;
  if (a->rows * blocks >= ((int64_t)1 << 31)) return fail(METIS_ERR_TOO_LARGE, "more rows than one launch takes");
  SampleParams p = {};
  p.logits = a->logits; p.ld = a->ld; p.vocab = (int32_t)a->vocab; p.each = (int32_t)each; p.dtype = a->dtype; p.u_64 = a->u_64 != 0; p.u = a->u;
  p.temperature = a->temperature; p.top_p = a->top_p; p.min_p = a->min_p; p.top_k = a->top_k;
  p.temperature_rows = a->temperature_rows; p.top_p_rows = a->top_p_rows; p.min_p_rows = a->min_p_rows; p.top_k_rows = a->top_k_rows;
  p.token = a->token; p.logprob = a->logprob;
  constexpr int kMostSmem = (2 * kBins + (METIS_SAMPLE_MAX_VOCAB / kMaxCluster / kThreads + 1) * kThreads) * 4;
  const bool half = a->dtype == METIS_DTYPE_BF16;
  METIS_CUDA_OK(half ? allow_smem<&sample_kernel<__nv_bfloat16>>(kMostSmem) : allow_smem<&sample_kernel<float>>(kMostSmem));
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(a->rows * blocks));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = (size_t)(2 * kBins + each * kThreads) * 4;
  cfg.stream = static_cast<cudaStream_t>(a->stream);
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)blocks;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = launch_overlap_enabled(kLaunchShort) ? 2 : 1;
  METIS_CUDA_OK(cudaLaunchKernelEx(&cfg, half ? sample_kernel<__nv_bfloat16> : sample_kernel<float>, p));
  count_rollout_launches(1);
  return METIS_OK;
}
