// One token for each row of logits: temperature, top-k, top-p, min-p, then the token at which the kept weights pass u times their sum.
//
//   w_i = exp((x_i - max x) (1/T)) in fp32 (1 at the maximum);  order: larger x first, equal ones by index
//   top-k keeps the first k of the order; top-p the shortest front of those whose weights are at least p of theirs; min-p those with w >= min_p.
//   Each keeps a front of the order, so that what is kept is "x above a cut, and the first n of those that equal it".
//
// A cluster of up to eight blocks takes a row: it is read once from memory, 16 bytes at a time, and stays in shared memory (in its type) for all passes.  Nothing is sorted; a cut is found by histograms:
//   bf16  The bins are the values themselves, from the largest one on: 4095 of them, those below 2^-8 in magnitude together in one.  That is every logit
//         within +-256.  A pass counts, five instructions and an addition in shared memory an element (the whole kernel runs 50); a bin's weight is its count times the
//         weight of its value, so that one histogram serves top-k, top-p and the sum of all.  (A cut in the bin of small values or behind the last one goes the other way.)
//   fp32  2048 bins of (max - x) / T in steps of 1/64, then 1024 at a time of the bits of the logits in the bin where the cut lies until one value is left.
//
// Whether a token is in or out goes by sums over up to all the vocabulary, and an fp32 sum would move borders with the order of its terms.  Here the
// sums have 64 bits: counts times weights; or, of fp32, a bin's weights lie within a factor of 2^(1/44), all 24 bits of each are multiples of one unit, and the
// bin adds them as whole numbers (two of at most 14 bits: 49664 of those fit 32 bits), exactly and in any order; bins, threads and blocks are
// added as doubles in a fixed order.  So a token does not depend on the schedule, and two programs that take the same weights find the same one.
#include "rollout.cuh"

#include <cooperative_groups.h>
#include <math_constants.h>

namespace cg = cooperative_groups;

namespace metis {
namespace {

constexpr int kThreads = 512;
constexpr int kBins = 2048;                        // of a histogram of weights: two words each
constexpr int kFine = 1024;                        // of one within a bin of those; what is in the bin is listed behind them
constexpr int kListed = 2 * kBins - 2 * kFine;
constexpr int kValues = 2 * kBins;                 // of a histogram of counts: one
constexpr int kMaxCluster = 8;
constexpr float kStep = 64.0f;                     // bins for a factor of e
constexpr int kLowBits = 13;

struct SampleParams {
  const void* logits;
  int64_t ld;
  int32_t vocab, each;                             // each: elements of a thread, an odd number of words (their reads then meet no bank twice)
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
struct Cut { float at; bool found; double ties; };        // kept are those above `at` and the first `ties` that equal it

struct Shared {
  double sums[kThreads / 32], more_sums[kThreads / 32];
  double gathered[2][kMaxCluster][2];
  Found found;
  Cut cut[2];                                      // of top-k, of top-p
  double share;                                    // weight of what top-k keeps
  uint32_t low, high, listed;                      // keys in the bin, of this block, and how many
  uint32_t maxima[kThreads / 32];
  uint32_t bins[2 * kBins];
};

// The same order as the numbers', as whole numbers; bf16 in 16 bits.
template <int kDrop> __device__ __forceinline__ uint32_t key_of(float x) {
  const uint32_t b = __float_as_uint(x);
  return ((b & 0x80000000u) ? ~b : b | 0x80000000u) >> kDrop;
}
template <int kDrop> __device__ __forceinline__ float value_of(uint32_t key) {
  const uint32_t k = key << kDrop;
  return __uint_as_float((k >> 31) ? k & 0x7fffffffu : ~(k | ((1u << kDrop) - 1u)));
}

// Elements in shared memory, in the type of the logits: NaN as -inf, -0 as 0.
template <typename T> struct Store;
template <> struct Store<float> {
  static constexpr int kDrop = 0, kWord = 1;        // bits that keys go without, elements of a 32-bit word
  static __device__ __forceinline__ float clean(float v) { return v == v ? v + 0.0f : -CUDART_INF_F; }
  static __device__ __forceinline__ uint32_t clean(uint32_t w) { return __float_as_uint(clean(__uint_as_float(w))); }
  static __device__ __forceinline__ float value(uint32_t w, int) { return __uint_as_float(w); }
};
template <> struct Store<__nv_bfloat16> {
  static constexpr int kDrop = 16, kWord = 2;
  static __device__ __forceinline__ uint32_t clean(uint32_t two) {
    const uint32_t lowest = 0xff80ff80u, none = 0u;                       // (the maximum of NaN and a number is the number)
    const __nv_bfloat162 v = __hadd2_rn(__hmax2(*reinterpret_cast<__nv_bfloat162*>(&two), *reinterpret_cast<const __nv_bfloat162*>(&lowest)), *reinterpret_cast<const __nv_bfloat162*>(&none));
    return *reinterpret_cast<const uint32_t*>(&v);
  }
  static __device__ __forceinline__ float value(uint32_t w, int half) { return half ? bf16_hi(w) : bf16_lo(w); }
  // two keys: negative ones with all bits turned, the others with the sign
  static __device__ __forceinline__ uint32_t keys(uint32_t w) {
    const uint32_t s = w & 0x80008000u;
    return w ^ ((s - (s >> 15)) | 0x80008000u);
  }
};
constexpr uint32_t kLowest16 = 0x007fu;            // the key of -inf
constexpr int kAbove = 0xbb80, kBelow = 0x447f;    // the keys of 2^-8 and -2^-8

// The cluster's blocks on one row.
template <typename T>
struct Row {
  using S = Store<T>;
  cg::cluster_group cluster;
  Shared& sh;
  const uint32_t* x;                               // this block's logits; -inf behind the last
  int blocks, rank, held;                          // held: elements of x
  float top, inverse;                              // the largest logit, 1/T
  int turn = 0;
  double own_small = 0.0;                          // weights that this block counted in the bin of small values

  __device__ float weight(float v) const { return v == top ? 1.0f : expf(__fmul_rn(__fsub_rn(v, top), inverse)); }

  // f(word) of each of the block's words, 16 bytes at a time
  template <typename F> __device__ __forceinline__ void each_word(const F& f) const {
#pragma unroll 2
    for (int i = threadIdx.x; i < held / S::kWord / 4; i += kThreads) {
      const uint4 w = reinterpret_cast<const uint4*>(x)[i];
      f(w.x); f(w.y); f(w.z); f(w.w);
    }
  }
  template <typename F> __device__ __forceinline__ void each(const F& f) const {
    each_word([&](uint32_t w) {
#pragma unroll
      for (int h = 0; h < S::kWord; ++h) f(S::value(w, h));
    });
  }

  // Two values of each block to all; two buffers in turn, so that one barrier does for both writing and reading.
  __device__ const double (*gather(double a, double b = 0.0))[2] {
    turn ^= 1;
    if (threadIdx.x < (unsigned)blocks) {
      double* to = cluster.map_shared_rank(&sh, threadIdx.x)->gathered[turn][rank];
      to[0] = a;
      to[1] = b;
    }
    cluster.sync();
    return sh.gathered[turn];
  }
  // What the blocks before this one have, and all.
  __device__ double ahead(double v, double& all) {
    const double (*g)[2] = gather(v);
    double before = 0.0;
    all = 0.0;
    for (int r = 0; r < blocks; ++r) {
      if (r == rank) before = all;
      all += g[r][0];
    }
    return before;
  }
  __device__ double sum_of(double mine) {
    double all;
    ahead(block_scan<kThreads>(mine, sh.sums).all, all);
    return all;
  }
  template <int N = kBins> __device__ void clear() {
    for (int i = threadIdx.x; i < 2 * N; i += kThreads) sh.bins[i] = 0u;
    __syncthreads();
  }

  // One word of all blocks' histograms, summed (all loads before the first addition: one from a peer takes some 700 cycles).
  __device__ uint32_t of_all(int word) const {
    uint32_t v[kMaxCluster], sum = 0;
#pragma unroll
    for (int r = 0; r < kMaxCluster; ++r) v[r] = r < blocks ? cluster.map_shared_rank(&sh, r)->bins[word] : 0u;
#pragma unroll
    for (int r = 0; r < kMaxCluster; ++r) sum += v[r];
    return sum;
  }

  __device__ uint64_t of_all_wide(int word) const {
    uint32_t v[kMaxCluster];
    uint64_t sum = 0;
#pragma unroll
    for (int r = 0; r < kMaxCluster; ++r) v[r] = r < blocks ? cluster.map_shared_rank(&sh, r)->bins[word] : 0u;
#pragma unroll
    for (int r = 0; r < kMaxCluster; ++r) sum += v[r];
    return sum;
  }

  // ---- histograms of weights (fp32; bf16 where the values' bins do not have the cut) ----

  __device__ int bin_of(float v) const {
    const float d = __fmul_rn(__fmul_rn(__fsub_rn(top, v), inverse), kStep);
    return v == top ? 0 : d < (float)(kBins - 1) ? (int)d : kBins - 1;
  }
  // The unit of a bin's weights is 2^unit_of: at least two bits below the last one of the smallest, e^(-(bin + 1) / 64) (log2(e) / 64 is below 1478 / 65536).  What
  // lies in the last bin, at most 2^-46 of the largest, loses what it has below 2^-72.
  __device__ static int unit_of(int bin) { return bin == kBins - 1 ? -72 : -(int)((uint32_t)(bin + 1) * 1478u >> 16) - 1 - 2 - 24; }
  __device__ static uint32_t whole(float w, int unit) { return (uint32_t)(w * __uint_as_float((uint32_t)(127 - unit) << 23)); }
  __device__ static double units(uint64_t m, int unit) { return (double)m * __hiloint2double((1023 + unit) << 20, 0); }

  template <bool kMass, int N> __device__ void add(int bin, float v, int unit) {
    if constexpr (kMass) {
      const uint32_t m = whole(weight(v), unit);
      atomicAdd(&sh.bins[bin], m & ((1u << kLowBits) - 1u));
      atomicAdd(&sh.bins[N + bin], m >> kLowBits);
    } else {
      atomicAdd(&sh.bins[bin], 1u);
    }
  }
  // Where the bins' sums, in order, reach the target; false if they do not.  unit: the bins', or their own where it is 1.  A negative target stands for that share of all.
  template <bool kMass, int N> __device__ bool reach(double& target, int unit, Found& out, double& all) {
    cluster.sync();
    constexpr int kMost = N / kThreads;
    const int slice = N / blocks, mine = slice > kThreads ? slice / kThreads : 1;
    double v[kMost], sum = 0.0;
#pragma unroll
    for (int i = 0; i < kMost; ++i) {
      const int local = threadIdx.x * mine + i;
      v[i] = 0.0;
      if (i >= mine || local >= slice) continue;
      const int bin = rank * slice + local;
      // (each block's word is below 2^29.6, and eight of them below 2^32 only where they are counts)
      uint64_t m;
      if constexpr (kMass) m = of_all_wide(bin) + (of_all_wide(N + bin) << kLowBits);
      else m = of_all(bin);
      if (m) v[i] = kMass ? units(m, unit == 1 ? unit_of(bin) : unit) : (double)m;
      sum += v[i];
    }
    const Scan<double> s = block_scan<kThreads>(sum, sh.sums);
    const double base = ahead(s.all, all);
    if (target < 0.0) target = fmax(-target * all, 1e-300);
    if (all < target) return false;                // the same for all blocks
    const double before = base + s.before, upto = base + s.upto;
    if (before < target && target <= upto) {
      Found f = {before, 0.0, 0};
      double next = before;
#pragma unroll
      for (int i = 0; i < kMost; ++i) {
        // (the last one that has anything, where rounding keeps the sum below the target)
        if (v[i] == 0.0 || (f.inside > 0.0 && target <= next)) continue;
        f = {next, v[i], rank * slice + (int)threadIdx.x * mine + i};
        next += v[i];
      }
      for (int r = 0; r < blocks; ++r) cluster.map_shared_rank(&sh, r)->found = f;
    }
    cluster.sync();
    out = sh.found;
    return true;
  }

  // The cut of the elements above `floor`: `at` such that the weights (or the number) of those above it are below the target and with those that equal
  // it are not; what is above, how many equal it, and the sum of all.  False if all of them do not reach the target; a negative one is a share of all, and comes back as
  // what that is.
  template <bool kMass> __device__ __forceinline__ bool cut(double& target, float floor, float& at, double& above, double& ties, double& all) {
    clear();
    each([&](float v) {
      if (v > floor) {
        const int bin = bin_of(v);
        add<kMass, kBins>(bin, v, kMass ? unit_of(bin) : 0);
      }
    });
    if (threadIdx.x == 0) { sh.low = 0xffffffffu; sh.high = 0u; sh.listed = 0u; }
    Found f;
    if (!reach<kMass, kBins>(target, 1, f, all)) return false;
    above = f.above;
    const int bin = f.bin, unit = unit_of(bin);
    // The bin's smallest and largest keys, and a list of them as long as there is room: levels go through that in place of the row (256 rows of 151936 fp32 logits,
    // top-p 0.95: 441 us without, 367 so; one row 43.5 and 36.4).
    uint32_t* const list = sh.bins + 2 * kFine;
    uint32_t low = 0xffffffffu, high = 0u;
    each([&](float v) {
      if (v > floor && bin_of(v) == bin) {
        const uint32_t k = key_of<S::kDrop>(v), n = atomicAdd(&sh.listed, 1u);
        if (n < (uint32_t)kListed) list[n] = k;
        low = min(low, k);
        high = max(high, k);
      }
    });
    low = __reduce_min_sync(0xffffffffu, low);
    high = __reduce_max_sync(0xffffffffu, high);
    if ((threadIdx.x & 31) == 0) { atomicMin(&sh.low, low); atomicMax(&sh.high, high); }
    __syncthreads();
    const int listed = (int)sh.listed;
    const double (*g)[2] = gather((double)sh.low, (double)sh.high);
    for (int r = 0; r < blocks; ++r) {
      low = min(low, (uint32_t)g[r][0]);
      high = max(high, (uint32_t)g[r][1]);
    }
    while (true) {
      const uint32_t span = high - low;
      const int shift = max(0, 22 - __clz(span));          // (span >> shift) < kFine
      clear<kFine>();
      auto member = [&](uint32_t k) {
        if (k >= low && k <= high) add<kMass, kFine>((int)((high - k) >> shift), value_of<S::kDrop>(k), unit);
      };
      if (listed <= kListed) {
        for (int i = threadIdx.x; i < listed; i += kThreads) member(list[i]);
      } else {
        each([&](float v) {
          if (v > floor && bin_of(v) == bin) member(key_of<S::kDrop>(v));
        });
      }
      // (a target that rounding puts in front of the bin's first element, or behind its last, is met by that one)
      Found next;
      double left = fmax(fmin(target - above, f.inside), 1e-300), of_bin;
      if (!reach<kMass, kFine>(left, unit, next, of_bin)) return false;
      above += next.above;
      f.inside = next.inside;
      high -= (uint32_t)next.bin << shift;
      if (shift == 0) break;
      low = max(low, high - ((1u << shift) - 1u));
    }
    at = value_of<S::kDrop>(high);
    ties = kMass ? rint(f.inside / units(whole(weight(at), unit), unit)) : f.inside;
    return true;
  }

  // of those that equal the cut, as many as have less than the target in front of them
  __device__ double ties_below(double target, double before, float at, double limit) const {
    const double w = (double)weight(at);
    double n = w > 0.0 ? fmax(1.0, ceil((target - before) / w)) : limit;
    while (n < limit && before + n * w < target) n += 1.0;
    while (n > 1.0 && before + (n - 1.0) * w >= target) n -= 1.0;
    return fmin(n, limit);
  }

  // Top-k and top-p by these histograms.  all_weights: of the whole row; where it is not known (0) and the nucleus is one of all, it comes out of the histogram: a pass over the row
  // less, 256 rows of 151936 fp32 logits 489 -> 440 us.  (A function of its own, for the registers of the way that needs none of it; by a
  // copy of the row, whose members would come from memory for every element.)
  static __device__ __noinline__ Cut by_weights(Row r, int64_t k, int64_t vocab, double top_p, double* all_weights, int* turn) {
    Cut c = {-CUDART_INF_F, false, 0.0};
    double above = 0.0;
    if (k > 0 && k < vocab) {
      float at;
      double want = (double)k, equal, all;
      if (r.cut<false>(want, -CUDART_INF_F, at, above, equal, all)) c = {at, true, (double)k - above};       // (else there are not so many)
    }
    if (top_p < 1.0) {
      double total = *all_weights, over = 0.0;
      if (c.found) {
        double sum = 0.0;
        r.each([&](float v) { if (v > c.at) sum += (double)r.weight(v); });
        over = r.sum_of(sum);
        total = over + c.ties * (double)r.weight(c.at);
      }
      const bool share = !c.found && total == 0.0 && top_p > 0.0;
      double target = share ? -top_p : fmax(top_p * total, 1e-300);       // (the first one is always kept)
      float at;
      double before, equal, all;
      const bool reached = r.cut<true>(target, c.at, at, before, equal, all);
      if (share) *all_weights = all;
      if (reached) c = {at, true, r.ties_below(target, before, at, equal)};
      else if (c.found) c.ties = r.ties_below(target, over, c.at, c.ties);  // all that are above the cut of top-k, and some that equal it
    }
    *turn = r.turn;
    return c;
  }

  // ---- the histogram of values (bf16) ----

  // Bins in the order of the values: bin 0 is the largest one's.  With d its distance to that one in keys, small = the bin of all that are below 2^-8 in magnitude
  // (if the largest is not below those) and gap = how many keys that bin swallows:
  //   keys above: d;   in it: small;   below: d - gap
  struct Values { int top, small, gap; bool has_small; };
  __device__ static Values values(int top) {
    if (top >= kAbove) return {top, top - kAbove + 1, kAbove - kBelow - 2, true};
    if (top > kBelow) return {top, 0, top - kBelow - 1, true};
    return {top, 0, 0, false};
  }

  // What this block has above a cut that by_values found, out of its own bins, and how many equal it; false where bins of several values would have to be told apart.
  template <typename Kept> __device__ bool own_above(float at, bool any_weight, const Kept& kept_weight, double& sum, double& equal) const {
    const Values b = values((int)key_of<16>(top));
    const int d = b.top - (int)key_of<16>(at), cut_bin = max(min(d, b.small), max(d, b.gap) - b.gap);
    const bool with_small = b.has_small && b.small < cut_bin;
    if (with_small && !any_weight) return false;
    sum = with_small && threadIdx.x == 0 ? own_small : 0.0;
    for (int bin = threadIdx.x; bin < cut_bin; bin += kThreads) {
      const uint32_t n = sh.bins[bin];
      if (n == 0 || (with_small && bin == b.small)) continue;
      sum += (double)n * kept_weight(value_of<16>((uint32_t)(b.top - bin - (bin > b.small ? b.gap : 0))));
    }
    equal = (double)sh.bins[cut_bin];
    return true;
  }

  // The same cut from counts; false where it lies in a bin of several values.  all_weights: of the row.
  __device__ bool by_values(int64_t k, double top_p, Cut& c, double& all_weights) {
    const Values b = values((int)key_of<16>(top));
    clear();
    double extra = 0.0;                            // weights in the bins of several values: the last one's, and the small ones'
    double extra_small = 0.0;
    // Two elements at a time: their keys are at most the largest one's, so that one subtraction serves both.  Those in bins of several values, and -inf
    // (which is in no bin), are found by comparing the values and go one by one.
    const uint32_t top2 = (uint32_t)b.top * 0x10001u, small2 = (uint32_t)b.small * 0x10001u, gap2 = (uint32_t)b.gap * 0x10001u;
    const int last_key = b.top - (kValues - 1) - (kValues - 1 > b.small ? b.gap : 0);
    const __nv_bfloat162 last_value = __float2bfloat162_rn(value_of<16>((uint32_t)max(last_key, (int)kLowest16))), tiny = __float2bfloat162_rn(b.has_small ? 0x1p-8f : 0.0f);
    each_word([&](uint32_t w) {
      const uint32_t d = top2 - S::keys(w), bin = __vmaxu2(__vminu2(d, small2), __vmaxu2(d, gap2) - gap2);
      const __nv_bfloat162 v = *reinterpret_cast<const __nv_bfloat162*>(&w);
      const uint32_t far = __hle2_mask(v, last_value), small = __hlt2_mask(__habs2(v), tiny);
      if ((far | small) == 0u) {
        atomicAdd(&sh.bins[bin & 0xffffu], 1u);
        atomicAdd(&sh.bins[bin >> 16], 1u);
        return;
      }
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const float x_h = S::value(w, h);
        const uint32_t half = 0xffffu << (16 * h);
        if (x_h == -CUDART_INF_F) continue;
        atomicAdd(&sh.bins[(far & half) ? kValues - 1 : (bin & half) >> (16 * h)], 1u);
        if (far & half) extra += (double)weight(x_h);
        else if (small & half) extra_small += (double)weight(x_h);
      }
    });
    // (sums of nothing, mostly)
    double rest = 0.0, small = 0.0;
    if (__syncthreads_or(extra != 0.0 || extra_small != 0.0)) {
      Scan<double> of_rest, of_small;
      block_scan_two<kThreads>(extra, extra_small, sh.sums, sh.more_sums, of_rest, of_small);
      rest = of_rest.all;
      small = own_small = of_small.all;
    }
    {
      const double (*g)[2] = gather(rest, small);  // (and the counts are there)
      rest = small = 0.0;
      for (int r = 0; r < blocks; ++r) { rest += g[r][0]; small += g[r][1]; }
    }
    // a thread has neighbouring bins: counts and weights, and what is before them
    constexpr int kMost = kValues / kThreads;
    const int slice = kValues / blocks, mine = slice / kThreads > 0 ? slice / kThreads : 1;
    const bool active = (int)threadIdx.x * mine < slice;
    const int first = rank * slice + (int)threadIdx.x * mine;
    uint32_t n[kMost];
    double count = 0.0, mass = 0.0;
    auto several = [&](int bin) { return bin == kValues - 1 || (b.has_small && bin == b.small); };
    auto value = [&](int bin) { return value_of<16>((uint32_t)(b.top - bin - (bin > b.small ? b.gap : 0))); };
    auto bin_mass = [&](int bin, uint32_t m) { return m == 0 ? 0.0 : bin == kValues - 1 ? rest : several(bin) ? small : (double)m * (double)weight(value(bin)); };
#pragma unroll
    for (int i = 0; i < kMost; ++i) {
      n[i] = 0;
      if (i >= mine || !active) continue;
      n[i] = of_all(first + i);
    }
#pragma unroll
    for (int i = 0; i < kMost; ++i) {
      if (n[i] == 0) continue;
      count += (double)n[i];
      mass += bin_mass(first + i, n[i]);
    }
    Scan<double> sc, sm;
    block_scan_two<kThreads>(count, mass, sh.sums, sh.more_sums, sc, sm);
    const double (*g)[2] = gather(sc.all, sm.all);
    double before_count = 0.0, before_mass = 0.0, all_count = 0.0;
    all_weights = 0.0;
    for (int r = 0; r < blocks; ++r) {
      if (r == rank) { before_count = all_count; before_mass = all_weights; }
      all_count += g[r][0];
      all_weights += g[r][1];
    }
    const double upto_count = before_count + sc.upto, upto_mass = before_mass + sm.upto;
    before_count += sc.before;
    before_mass += sm.before;
    // (ties of -1: the cut lies in a bin of several values)
    c = {-CUDART_INF_F, false, 0.0};
    double total = all_weights;
    if (k > 0 && (double)k < all_count) {
      const double want = (double)k;
      if (before_count < want && want <= upto_count) {
        Cut found = {0.0f, true, -1.0};
        double ahead_n = before_count, ahead_m = before_mass, share = 0.0;
#pragma unroll
        for (int i = 0; i < kMost; ++i) {
          if (n[i] == 0) continue;
          if (ahead_n < want && want <= ahead_n + (double)n[i] && !several(first + i)) {
            found = {value(first + i), true, want - ahead_n};
            share = ahead_m + found.ties * (double)weight(found.at);
          }
          ahead_n += (double)n[i];
          ahead_m += bin_mass(first + i, n[i]);
        }
        for (int r = 0; r < blocks; ++r) {
          Shared* peer = cluster.map_shared_rank(&sh, r);
          peer->cut[0] = found;
          peer->share = share;
        }
      }
      cluster.sync();
      c = sh.cut[0];
      if (c.ties < 0.0) return false;
      total = sh.share;
    }
    if (top_p < 1.0) {
      const double target = fmax(top_p * total, 1e-300);                  // (the first one is always kept)
      if (before_mass < target && target <= upto_mass) {
        Cut found = {0.0f, true, -1.0};
        double ahead_m = before_mass;
        bool open = true;
#pragma unroll
        for (int i = 0; i < kMost; ++i) {
          // (the last one that has anything, where rounding keeps the sum below the target)
          if (n[i] == 0 || !open) continue;
          const double m = bin_mass(first + i, n[i]);
          if (m == 0.0) continue;
          found = {value(first + i), true, several(first + i) ? -1.0 : ties_below(target, ahead_m, value(first + i), (double)n[i])};
          open = ahead_m + m < target;
          ahead_m += m;
        }
        if (c.found && found.ties >= 0.0 && (found.at < c.at || (found.at == c.at && found.ties > c.ties))) found = c;
        for (int r = 0; r < blocks; ++r) cluster.map_shared_rank(&sh, r)->cut[1] = found;
      }
      cluster.sync();
      c = sh.cut[1];
      if (c.ties < 0.0) return false;
    }
    return true;
  }
};

template <typename T>
__global__ void __launch_bounds__(kThreads, 2) sample_kernel(const SampleParams p) {
  using S = Store<T>;
  extern __shared__ __align__(16) uint32_t x[];
  __shared__ Shared sh;
  const cg::cluster_group cluster = cg::this_cluster();
  const int blocks = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
  const int64_t row = blockIdx.x / blocks;
  const int held = p.each * kThreads, first = rank * held, here = max(0, min(held, p.vocab - first));
  cluster.barrier_arrive();                        // (a block is written to by the others once all have begun)
  grid_dependency_wait();

  const float t = p.temperature_rows ? p.temperature_rows[row] : p.temperature, min_p = p.min_p_rows ? p.min_p_rows[row] : p.min_p;
  const double top_p = p.top_p_rows ? (double)p.top_p_rows[row] : p.top_p;
  int64_t k = p.top_k_rows ? p.top_k_rows[row] : p.top_k;
  const double u = p.u_64 ? static_cast<const double*>(p.u)[row] : (double)static_cast<const float*>(p.u)[row];

  // ---- the row; NaN and what is behind it as -inf, -0 as 0 ----
  const T* from = static_cast<const T*>(p.logits) + row * p.ld + first;
  constexpr int kWide = 16 / (int)sizeof(T);
  const int wide = (reinterpret_cast<uintptr_t>(from) & 15) == 0 ? here / kWide : 0;
  float most = -CUDART_INF_F;
  uint32_t most_two = 0xff80ff80u;                 // of the even elements, of the odd ones
  auto track = [&](uint32_t w) {
    if constexpr (sizeof(T) == 2) {
      const __nv_bfloat162 v = __hmax2(*reinterpret_cast<__nv_bfloat162*>(&most_two), *reinterpret_cast<__nv_bfloat162*>(&w));
      most_two = *reinterpret_cast<const uint32_t*>(&v);
    } else {
      most = fmaxf(most, __uint_as_float(w));
    }
  };
#pragma unroll 4
  for (int i = threadIdx.x; i < wide; i += kThreads) {
    const uint4 v = __ldcs(reinterpret_cast<const uint4*>(from) + i);
    const uint4 w = make_uint4(S::clean(v.x), S::clean(v.y), S::clean(v.z), S::clean(v.w));
    track(w.x); track(w.y); track(w.z); track(w.w);
    reinterpret_cast<uint4*>(x)[i] = w;
  }
  for (int i = wide * kWide + threadIdx.x; i < held; i += kThreads) {
    if constexpr (sizeof(T) == 2) {
      const uint32_t w = S::clean(i < here ? 0xff800000u | reinterpret_cast<const uint16_t*>(from)[i] : 0xff80ff80u);
      track(w);
      reinterpret_cast<uint16_t*>(x)[i] = (uint16_t)w;
    } else {
      const uint32_t w = i < here ? S::clean(__float_as_uint(from[i])) : 0xff800000u;
      track(w);
      x[i] = w;
    }
  }
  if constexpr (sizeof(T) == 2) most = fmaxf(bf16_lo(most_two), bf16_hi(most_two));
  uint32_t best = key_of<S::kDrop>(most);          // the largest key
  best = __reduce_max_sync(0xffffffffu, best);
  if ((threadIdx.x & 31) == 0) sh.maxima[threadIdx.x >> 5] = best;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kThreads / 32; ++w) best = max(best, sh.maxima[w]);

  cluster.barrier_wait();
  Row<T> r{cluster, sh, x, blocks, rank, held, 0.0f, 0.0f};
  {
    const double (*g)[2] = r.gather((double)best);
    for (int i = 0; i < blocks; ++i) best = max(best, (uint32_t)g[i][0]);
  }
  const float top = value_of<S::kDrop>(best);
  const bool fine = (t == 0.0f || (t >= 0x1p-126f && t <= 3.4028235e38f)) && top_p >= 0.0 && top_p <= 1.0 && min_p >= 0.0f && min_p <= 1.0f && k >= 0 && u >= 0.0 && u < 1.0 &&
                    top > -CUDART_INF_F;
  if (!fine) {                                     // (for all blocks of the cluster)
    if (rank == 0 && threadIdx.x == 0) {
      p.token[row] = -1;
      if (p.logprob) p.logprob[row] = CUDART_NAN_F;
    }
    return;
  }
  const float heat = t == 0.0f ? 1.0f : t;
  if (t == 0.0f) k = 1;
  r.top = top;
  r.inverse = __fdiv_rn(1.0f, heat);

  // ---- the cut, and the weight of all ----
  Cut cut = {-CUDART_INF_F, false, 0.0};
  double all_weights = 0.0;
  const bool filtered = k != 1 && ((k > 0 && k < p.vocab) || top_p < 1.0), everything = k == 0 && !filtered && min_p == 0.0f;
  bool settled = !filtered, counted = false;
  if constexpr (sizeof(T) == 2)
    if (filtered) {
      settled = r.by_values(k, top_p, cut, all_weights);
      counted = true;
    }
  // (a nucleus of all, without top-k, finds it by itself)
  const bool found_later = !settled && top_p > 0.0 && top_p < 1.0 && !(k > 0 && k < p.vocab);
  if (!counted && !everything && !found_later && (p.logprob || (filtered && top_p < 1.0))) {
    double sum = 0.0;
    r.each([&](float v) { sum += (double)r.weight(v); });
    all_weights = r.sum_of(sum);
  }
  if (!settled) cut = Row<T>::by_weights(r, k, p.vocab, top_p, &all_weights, &r.turn);
  if (k == 1) cut = {top, true, 1.0};

  // ---- the kept weights of this thread's elements, in order of their indices ----
  const float from_value = cut.found ? cut.at : sizeof(T) == 2 ? -0x1.fep127f : -3.4028235e38f;  // (the lowest finite one: -inf is never kept)
  const int words = p.each / S::kWord, from_word = threadIdx.x * words;
  auto walk = [&](const auto& f) {                 // f(index, value) of each that is not below the cut
    __nv_bfloat162 from_two = __float2bfloat162_rn(from_value);
    for (int w = from_word; w < from_word + words; ++w) {
      uint32_t v = x[w];
      if constexpr (sizeof(T) == 4) {
        if (__uint_as_float(v) >= from_value && !f(w, __uint_as_float(v))) return;
      } else {
        const uint32_t in = __hge2_mask(*reinterpret_cast<__nv_bfloat162*>(&v), from_two);
        if (in == 0u) continue;
        if ((in & 0xffffu) && !f(2 * w, bf16_lo(v))) return;
        if ((in >> 16) && !f(2 * w + 1, bf16_hi(v))) return;
      }
    }
  };
  auto kept_weight = [&](float v) {
    const float w = r.weight(v);
    return w >= min_p ? (double)w : 0.0;
  };
  // this thread's above the cut, summed, and those that equal it, counted
  double sum = 0.0;
  int32_t equal = 0;
  auto count_in = [&](float v) {
    if (cut.found && v == cut.at) ++equal; else sum += kept_weight(v);
  };
  auto count_own = [&]() {
    if (sizeof(T) == 2 && cut.found) {
      // Few are kept, and not the same ones in all lanes: 32 elements are compared first, two at a time into the bits of two words, and the lanes
      // then go through theirs (lanes that went through all elements together took 22 thousand cycles of a row's 80).
      const __nv_bfloat162 from_two = __float2bfloat162_rn(from_value);
      const uint16_t* const mine = reinterpret_cast<const uint16_t*>(x + from_word);
      for (int w = 0; w < words; w += 16) {
        uint32_t in[2] = {0u, 0u};                   // of word j: bit 2 j for its low half, 17 + 2 j for the other
#pragma unroll
        for (int j = 0; j < 16; ++j)
          if (w + j < words) {
            const uint32_t v = x[from_word + w + j];
            in[j / 8] |= __hge2_mask(*reinterpret_cast<const __nv_bfloat162*>(&v), from_two) & (0x00020001u << (2 * (j % 8)));
          }
        while (in[0] | in[1]) {
          const bool second = in[0] == 0u;
          const uint32_t bits = second ? in[1] : in[0], rest = bits & (bits - 1u);
          const int at = __ffs(bits) - 1, element = (at & 15) + (second ? 16 : 0);         // (17 + 2 j, less 16, is 2 j + 1)
          if (second) in[1] = rest; else in[0] = rest;
          count_in(__uint_as_float((uint32_t)mine[2 * w + element] << 16));
        }
      }
    } else {
#pragma unroll 4
      for (int w = from_word; w < from_word + words; ++w) {
        const uint32_t v = x[w];
#pragma unroll
        for (int h = 0; h < S::kWord; ++h)
          if (S::value(v, h) >= from_value) count_in(S::value(v, h));
      }
    }
  };
  // Which block has the mark goes by the blocks' sums, the same numbers in all of them; there, a thread by its own.  Where there are counts of this block's values its
  // sum comes from those, a few hundred of them, and the elements are gone through by the block that has the mark alone, while the others leave (256 rows of 151936, top-p
  // 0.95: 144 us, 140 where they all go through theirs and leave, 132 so).
  double nth = 0.0, kept_ties = 0.0;               // ties before this thread's, and how many of its own are kept
  const double tie_weight = cut.found ? kept_weight(cut.at) : 0.0;
  double block_sum = 0.0, block_equal = 0.0;
  bool listed = false;
  if constexpr (sizeof(T) == 2)
    if (counted && settled && cut.found) {
      listed = r.own_above(cut.at, min_p == 0.0f, kept_weight, block_sum, block_equal);
      if (listed) block_sum = block_scan<kThreads>(block_sum, sh.sums).all;
    }
  if (!listed) {
    count_own();
    Scan<double> se, ss;
    block_scan_two<kThreads>((double)equal, sum, sh.sums, sh.more_sums, se, ss);
    nth = se.before;
    block_sum = ss.all;
    block_equal = se.all;
  }
  // (Behind this last exchange no block reads or writes what another one has: those that are done leave, and make room for other rows.)
  double total = 0.0, base = 0.0, upto = 0.0, ties_ahead = 0.0;
  {
    const double (*g)[2] = r.gather(block_equal, block_sum);
    double ties_before = 0.0;
    for (int i = 0; i < blocks; ++i) {
      if (i == rank) { base = total; ties_ahead = ties_before; }
      total += g[i][1] + fmin(fmax(cut.ties - ties_before, 0.0), g[i][0]) * tie_weight;
      ties_before += g[i][0];
      if (i == rank) upto = total;
    }
  }
  if (everything) all_weights = total;
  double mark = u * total;
  if (mark >= total) mark = __longlong_as_double(__double_as_longlong(total) - 1);      // (rounded up: the last one)
  if (base <= mark && mark < upto) {               // (one block of the cluster)
    if (listed) {
      count_own();
      // (where all or none of the block's ties are kept, it is the same for each thread)
      if (ties_ahead < cut.ties && cut.ties < ties_ahead + block_equal) nth = block_scan<kThreads>((double)equal, sh.sums).before;
    }
    nth += ties_ahead;
    kept_ties = fmin(fmax(cut.ties - nth, 0.0), (double)equal);
    sum += kept_ties * tie_weight;
    const Scan<double> s = block_scan<kThreads>(sum, sh.sums);
    mark -= base;
    if (mark >= s.all) mark = __longlong_as_double(__double_as_longlong(s.all) - 1);    // (the sums of threads and of blocks are rounded apart)
    if (s.before <= mark && mark < s.upto) {
      double acc = s.before;
      int token = -1;
      float chosen = 0.0f;
      walk([&](int i, float v) {
        if (cut.found && v == cut.at) {
          nth += 1.0;
          if (nth > cut.ties) return true;
        }
        const double w = kept_weight(v);
        if (w == 0.0) return true;
        acc += w;
        token = i;
        chosen = v;
        return acc <= mark;
      });
      p.token[row] = first + token;
      if (p.logprob) p.logprob[row] = (float)((chosen == top ? 0.0 : ((double)chosen - (double)top) / (double)heat) - log(all_weights));
    }
  }
}

}  // namespace
}  // namespace metis

using namespace metis;

extern "C" int32_t metis_sample(const metis_sample_args* a) {
  if (!a || !a->logits || !a->u || !a->token) return fail(METIS_ERR_BAD_ARGUMENT, "null pointer");
  if (a->dtype != METIS_DTYPE_BF16 && a->dtype != METIS_DTYPE_F32) return fail(METIS_ERR_BAD_ARGUMENT, "logits must be bf16 or fp32");
  if (a->rows <= 0 || a->vocab <= 0 || (a->rows > 1 && a->ld < a->vocab)) return fail(METIS_ERR_BAD_SHAPE, "rows and vocab must be positive, rows of logits apart");
  if (a->vocab > METIS_SAMPLE_MAX_VOCAB) return fail(METIS_ERR_TOO_LARGE, "vocabularies have at most %d entries", METIS_SAMPLE_MAX_VOCAB);
  const bool half = a->dtype == METIS_DTYPE_BF16;
  // A block for each 8192 entries up to eight of them while the GPU holds all rows at once (two blocks an SM); of more rows fewer and larger ones, of up to
  // 96 KB each: few are sooner done, more blocks wait longer for one another.
  int blocks = 1;
  while (blocks < kMaxCluster && a->vocab > (int64_t)blocks * 8192 && (a->rows * blocks * 2 <= (int64_t)device_sm_count() * 2 || a->vocab > (int64_t)blocks * (half ? 49152 : 24576))) blocks *= 2;
  const int word = half ? 2 : 1;
  const int64_t each = (ceil_div(ceil_div(a->vocab, blocks), (int64_t)kThreads * word) | 1) * word;
  if (a->rows * blocks >= ((int64_t)1 << 31)) return fail(METIS_ERR_TOO_LARGE, "more rows than one launch takes");
  SampleParams p = {};
  p.logits = a->logits; p.ld = a->ld; p.vocab = (int32_t)a->vocab; p.each = (int32_t)each; p.u_64 = a->u_64 != 0; p.u = a->u;
  p.temperature = a->temperature; p.top_p = a->top_p; p.min_p = a->min_p; p.top_k = a->top_k;
  p.temperature_rows = a->temperature_rows; p.top_p_rows = a->top_p_rows; p.min_p_rows = a->min_p_rows; p.top_k_rows = a->top_k_rows;
  p.token = a->token; p.logprob = a->logprob;
  constexpr int kMostSmem = (METIS_SAMPLE_MAX_VOCAB / kMaxCluster / kThreads + 1) * kThreads * 4;
  METIS_CUDA_OK(half ? allow_smem<&sample_kernel<__nv_bfloat16>>(kMostSmem) : allow_smem<&sample_kernel<float>>(kMostSmem));
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(a->rows * blocks));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = (size_t)each * kThreads * (half ? 2 : 4);
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
