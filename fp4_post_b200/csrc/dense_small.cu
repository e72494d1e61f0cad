// The bf16 products of dense_gemm.cu for few tokens (sm_100a): the weight is what has to be read, and the read is what bounds them.
//
// Rows of the weight are the 128-row operand of the tensor core and tokens its columns, D[weight row, token]: the weight streams through
// shared memory once, in the order it lies in, and the tensor core's time is that of 16 to 128 columns.
//
//   linear   a cluster takes a tile of 32, 64 or 128 weight rows and its CTAs share the contraction; their partial sums meet in
//            distributed shared memory, where each CTA adds a part of the tile in rank order and applies the epilogue.  One launch.
//   stats    (the head's losses) a CTA takes an even part of the vocabulary, in units of 32 rows, tile after tile with two accumulators;
//            every epilogue lane keeps running statistics for each token of the rows it sees and the lanes are merged at the end.
//
// Roles: warp 0 loads, warp 1 issues, warps 2 and up drain tensor memory.  No copy is multicast; every wait is bounded.
#include "dense.cuh"
#include "pair.cuh"

namespace metis {

constexpr int kSmallThreads = 384;                       // loader, issuer, eight that drain tensor memory; the epilogue is everybody's
// Shared memory of a CTA: two fit an SM, so that clusters of any size find room; one where all CTAs run at once and leave none idle.
constexpr int kSmallBudget = 100 * 1024, kSmallBudgetAlone = 200 * 1024, kStatsBudget = 200 * 1024;

// Barriers, tensor memory and the abort flag behind the pipeline's stages.
struct SmallBars {
  uint64_t *full, *empty, *acc_full, *acc_empty, *drain;
  uint32_t* tmem_slot;
  volatile int* abort_flag;
  __device__ __forceinline__ SmallBars(uint8_t* at, int stages) {
    full = reinterpret_cast<uint64_t*>(at);
    empty = full + stages;
    acc_full = empty + stages;                             // [2]
    acc_empty = acc_full + 2;                              // [2]
    drain = acc_empty + 2;
    tmem_slot = reinterpret_cast<uint32_t*>(drain + 1);
    abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  }
};

__device__ __forceinline__ void small_setup(const SmallBars& b, int stages, uint32_t tmem_cols, int epilogue_warps) {
  if (threadIdx.x == 0) {
    for (int s = 0; s < stages; ++s) { mbar_init(&b.full[s], 1); mbar_init(&b.empty[s], 1); }
    for (int i = 0; i < 2; ++i) { mbar_init(&b.acc_full[i], 1); mbar_init(&b.acc_empty[i], epilogue_warps); }
    mbar_init(b.drain, 1);
    *b.abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  if ((threadIdx.x >> 5) == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(b.tmem_slot)), "r"(tmem_cols) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
}
__device__ __forceinline__ void small_free(uint32_t tmem_base, uint32_t tmem_cols) {
  if ((threadIdx.x >> 5) == 1) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(tmem_cols) : "memory");
  }
}
// tensor-memory columns for `cols` (a power of two, at least what one load reads)
__host__ __device__ static inline uint32_t small_tmem_cols(int cols) { return cols <= 32 ? 32u : cols <= 64 ? 64u : cols <= 128 ? 128u : 256u; }

__device__ __forceinline__ float4 load_cluster_f32x4(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ float load_cluster_f32(uint32_t addr) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
  return v;
}
// Eight elements of a row of a bf16 operand as words: together (vec: 16-byte aligned rows), or `apart` from one another; those past the end
// of the row are zero.
__device__ __forceinline__ void load_row8(const __nv_bfloat16* src, bool vec, int apart, int64_t left, uint32_t (&w)[4]) {
  if (vec && left >= 8) {
    const uint4 q = *reinterpret_cast<const uint4*>(src);
    w[0] = q.x; w[1] = q.y; w[2] = q.z; w[3] = q.w;
  } else {
    const unsigned short* s = reinterpret_cast<const unsigned short*>(src);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t lo = 2 * i * apart < left ? s[2 * i * apart] : 0, hi = (2 * i + 1) * apart < left ? s[(2 * i + 1) * apart] : 0;
      w[i] = lo | (hi << 16);
    }
  }
}
__device__ __forceinline__ void store_words8(unsigned short* dst, bool vec, int apart, int64_t left, const uint32_t (&w)[4]) {
  if (vec && left >= 8) {
    *reinterpret_cast<uint4*>(dst) = make_uint4(w[0], w[1], w[2], w[3]);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) if (i * apart < left) dst[i * apart] = (unsigned short)(w[i >> 1] >> ((i & 1) * 16));
  }
}
__device__ __forceinline__ void store_row8(__nv_bfloat16* dst, bool vec, int apart, int64_t left, const float (&v)[8]) {
  const uint32_t w[4] = {pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3]), pack_bf16(v[4], v[5]), pack_bf16(v[6], v[7])};
  store_words8(reinterpret_cast<unsigned short*>(dst), vec, apart, left, w);
}

// One stage's MMAs: D[128 weight rows, bn tokens] += weights [128, 64] tokens [bn, 64]^T.  A tile of fewer than 128 rows reads what lies
// behind it in shared memory for the others; those lanes of the accumulator are not used.
template <bool kWMn>
__device__ __forceinline__ void small_mma(uint32_t d_tmem, uint32_t sw, uint32_t st, uint32_t idesc, bool first) {
  constexpr uint32_t lead = kWMn ? (uint32_t)((64 * 128) >> 4) : 1u, step = kWMn ? (16u * 128u) >> 4 : 2u;
  const uint32_t w_lo = ((sw & 0x3FFFFu) >> 4) | (lead << 16), t_lo = operand_desc_lo(st);
#pragma unroll
  for (int j = 0; j < 4; ++j) tc_mma_bf16(d_tmem, w_lo + step * j, t_lo + 2 * j, kOperandDescHi, idesc, (!first || j > 0) ? 1u : 0u);
}

// kWMn: the weight lies with the contraction in its rows ([K, N], the gradient of an input)
template <bool kWMn>
__global__ void __launch_bounds__(kSmallThreads)
dense_small_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_t, const DenseParams p, const SmallShape sh) {
  extern __shared__ uint8_t smem_raw[];
  // the dynamic window starts at the same offset in all CTAs of the cluster: so does the partial sums' place
  uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  const int token_bytes = sh.bn * 128;
  const SmallBars bars(smem, sh.stages);
  uint8_t* pipe = smem + 1024;
  float* partial = reinterpret_cast<float*>(pipe);         // [bn][128], once the pipeline has run dry
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = sh.splits > 1 ? (int)cluster_ctarank() : 0;
  const int64_t tile = blockIdx.x / sh.splits;
  const int64_t n0 = tile * sh.rows, m0 = (int64_t)blockIdx.y * sh.bn;
  // this CTA's blocks of 64 along the contraction, `kb` of them to a stage (at least one: the host sees to it)
  const int blocks_all = (int)((p.K + 63) / 64);
  const int block0 = rank * sh.blocks_per_split;
  const int blocks = blocks_all - block0 < sh.blocks_per_split ? blocks_all - block0 : sh.blocks_per_split;
  const int block_bytes = token_bytes + sh.rows * 128;
  const int iters = (blocks + sh.kb - 1) / sh.kb;
  const uint32_t tmem_cols = small_tmem_cols(sh.bn);
  small_setup(bars, sh.stages, tmem_cols, 1);
  const uint32_t tmem_base = *bars.tmem_slot;
  grid_dependency_wait();

  if (warp == 0) {
    int stage = 0;
    uint32_t phase = 0;
    const uint32_t base = smem_u32(pipe);
    for (int it = 0; it < iters; ++it) {
      if (!__all_sync(0xffffffffu, mbar_wait(&bars.empty[stage], phase ^ 1u, bars.abort_flag))) {
        if (lane == 0) report(p.status, bars.abort_flag, METIS_DEV_TIMEOUT_MMA);
        break;
      }
      if (elect_one()) {
        const uint32_t bar = smem_u32(&bars.full[stage]);
        const int n_blocks = blocks - it * sh.kb < sh.kb ? blocks - it * sh.kb : sh.kb;
        mbar_expect_tx_addr(bar, (uint32_t)(n_blocks * block_bytes));
        for (int b = 0; b < n_blocks; ++b) {
          const uint32_t st = base + stage * sh.stage_bytes + b * block_bytes, sw = st + token_bytes;
          const int32_t k0 = (block0 + it * sh.kb + b) * 64;
          if (kWMn) {
            for (int r = 0; r < sh.rows; r += 64) tma_load_2d_addr(sw + r * 128, &map_w, (int32_t)n0 + r, k0, bar);
          } else {
            tma_load_2d_addr(sw, &map_w, k0, (int32_t)n0, bar);
          }
          tma_load_2d_addr(st, &map_t, k0, (int32_t)m0, bar);
        }
      }
      if (++stage == sh.stages) { stage = 0; phase ^= 1u; }
    }
    grid_launch_dependents();
  } else if (warp == 1) {
    int stage = 0;
    uint32_t phase = 0;
    bool ok = true, issued = false;
    const uint32_t base = smem_u32(pipe), idesc = idesc_bf16(sh.bn) | (kWMn ? (1u << 15) : 0u);
    for (int it = 0; it < iters; ++it) {
      ok = __all_sync(0xffffffffu, mbar_wait(&bars.full[stage], phase, bars.abort_flag));
      if (!ok) {
        if (lane == 0) report(p.status, bars.abort_flag, METIS_DEV_TIMEOUT_TMA);
        break;
      }
      tc_fence_after();
      if (elect_one()) {
        const int n_blocks = blocks - it * sh.kb < sh.kb ? blocks - it * sh.kb : sh.kb;
        for (int b = 0; b < n_blocks; ++b) {
          const uint32_t st = base + stage * sh.stage_bytes + b * block_bytes;
          small_mma<kWMn>(tmem_base, st + token_bytes, st, idesc, it == 0 && b == 0);
        }
        tc_commit(&bars.empty[stage]);
        if (it == iters - 1) tc_commit(bars.acc_full);
      }
      issued = true;
      if (++stage == sh.stages) { stage = 0; phase ^= 1u; }
    }
    if (!ok && issued && elect_one()) {
      tc_commit(bars.drain);
      const uint64_t t0 = global_ns();
      while (!mbar_try(bars.drain, 0) && global_ns() - t0 < kWaitLimitNs) {}
    }
    __syncwarp();
  } else if (warp < 10) {
    const int q = warp & 3;
    if (!mbar_wait(bars.acc_full, 0, bars.abort_flag)) {
      if (lane == 0) report(p.status, bars.abort_flag, METIS_DEV_TIMEOUT_MMA);
    } else {
      // every MMA has completed: the stages are free
      tc_fence_after();
      const uint32_t t_row = tmem_base + ((uint32_t)(q * 32) << 16);
      if (q * 32 < sh.rows) {
        for (int c0 = ((warp - 2) >> 2) * 32; c0 < sh.bn && m0 + c0 < p.M; c0 += 64) {
          uint32_t r[32];
          tc_load32(t_row + c0, r);
          tc_wait_ld(r);
#pragma unroll
          for (int i = 0; i < 32; ++i) if (c0 + i < sh.bn) partial[(c0 + i) * 128 + q * 32 + lane] = __uint_as_float(r[i]);
        }
      }
      tc_fence_before();
    }
  }
  tc_fence_before();
  __syncthreads();
  small_free(tmem_base, tmem_cols);
  if (sh.splits > 1) cluster_sync_all();                   // the partial sums of every CTA are in place

  // Items of eight elements of one token, the CTAs of the cluster in turn; a thread has the epilogue's operands of kFly items in
  // flight before it uses them (one element at a time, 64 tokens of the silu and gate of 18944 rows: 56 us for the product; 29 so).
  // The eight lie together where rows are 16-byte aligned, else an item apart, so that neighbouring lanes have neighbouring elements.
  const int tokens = p.half ? p.half_rows : p.M - m0 < sh.bn ? (int)(p.M - m0) : sh.bn;       // (two parts are one tile)
  const int shift = sh.rows == 128 ? 4 : sh.rows == 64 ? 3 : 2;        // log2 of the items of a token
  const bool wide = p.d_wide && (!p.gate || p.gate_wide) && (!p.residual || p.residual_wide);
  const int apart = wide ? 1 : 1 << shift, first = wide ? 8 : 1;
  const uint32_t mine = smem_u32(partial);
  constexpr int kFly = 4;
  const int step = sh.splits * kSmallThreads;
  for (int e0 = rank * kSmallThreads + threadIdx.x; e0 < tokens << shift; e0 += kFly * step) {
    uint32_t gate[kFly][4], residual[kFly][4];
#pragma unroll
    for (int k = 0; k < kFly; ++k) {
      const int e = e0 + k * step;
      const int64_t n = n0 + first * (e & ((1 << shift) - 1)), m = m0 + (e >> shift);
      if (e < tokens << shift && n < p.N) {
        if (p.gate) load_row8(p.gate + m * p.ldgate + n, wide, apart, p.N - n, gate[k]);
        if (p.residual) load_row8(p.residual + m * p.ldr + n, wide, apart, p.N - n, residual[k]);
      }
    }
#pragma unroll
    for (int k = 0; k < kFly; ++k) {
      const int e = e0 + k * step;
      const int r = first * (e & ((1 << shift) - 1)), t = e >> shift;
      const int64_t n = n0 + r, m = m0 + t, left = p.N - n;
      if (e >= tokens << shift || left <= 0) continue;
      float v[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = 0.0f;
      const uint32_t at = mine + (t * 128 + r) * 4;
#pragma unroll 4
      for (int s = 0; s < sh.splits; ++s) {
        const uint32_t from = sh.splits > 1 ? map_to_cta(at, s) : at;
        if (wide) {
          const float4 a = load_cluster_f32x4(from), b = load_cluster_f32x4(from + 16);
          v[0] += a.x; v[1] += a.y; v[2] += a.z; v[3] += a.w;
          v[4] += b.x; v[5] += b.y; v[6] += b.z; v[7] += b.w;
        } else {
#pragma unroll
          for (int i = 0; i < 8; ++i) v[i] += load_cluster_f32(from + i * apart * 4);
        }
        if (p.half) {                                      // (a product: rows of 16-byte pieces)
          const float4 a = load_cluster_f32x4(from + p.half * 512), b = load_cluster_f32x4(from + p.half * 512 + 16);
          v[0] += a.x; v[1] += a.y; v[2] += a.z; v[3] += a.w;
          v[4] += b.x; v[5] += b.y; v[6] += b.z; v[7] += b.w;
        }
      }
      if (p.bias) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int64_t c = n + i * apart;
          if (i * apart < left) v[i] += p.bias_f32 ? static_cast<const float*>(p.bias)[c] : __bfloat162float(static_cast<const __nv_bfloat16*>(p.bias)[c]);
        }
      }
      if (p.slope) {
        uint32_t slopes[4];
        activate_both_all(p.act, v, slopes);
        store_words8(reinterpret_cast<unsigned short*>(p.slope) + m * p.ldslope + n, wide, apart, left, slopes);
      } else {
        activate_all(p.act, v);
      }
      if (p.act_out) store_row8(p.act_out + m * p.ldact + n, wide, apart, left, v);
      if (p.gate) {
#pragma unroll
        for (int i = 0; i < 4; ++i) { v[2 * i] *= bf16_lo(gate[k][i]); v[2 * i + 1] *= bf16_hi(gate[k][i]); }
      }
      if (p.residual) {
#pragma unroll
        for (int i = 0; i < 4; ++i) { v[2 * i] += bf16_lo(residual[k][i]); v[2 * i + 1] += bf16_hi(residual[k][i]); }
      }
      store_row8(p.d + m * p.ldd + n, wide, apart, left, v);
    }
  }
  __syncwarp();
  if (sh.splits > 1) cluster_sync_all();                   // no CTA goes while another reads its shared memory
}

// ---- statistics of the head -------------------------------------------------------------------------------------

// Statistics of one more logit l (times log2 e): one exponential, of the smaller against the larger.  m starts at a finite value below
// every logit that is not -infinity.
constexpr float kNoLogit = -1e30f;
template <bool kEntropy> __device__ __forceinline__ void stats_add(float l, float& m, float& s, float& e) {
  const float d = l - m, x = exp2_fast(-fabsf(d));
  if (d > 0.0f) {
    if constexpr (kEntropy) e = x * fmaf(-d, s, e);
    s = fmaf(s, x, 1.0f);
    m = l;
  } else {
    if constexpr (kEntropy) e = fmaf(x, fmaxf(d, kNoLogit), e);
    s += x;
  }
}

// kWarps epilogue warps: four for each 32 tokens
template <bool kEntropy, int kWarps>
__global__ void __launch_bounds__(64 + 32 * kWarps, 1)
dense_small_stats_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_t, const DenseParams p, const SmallShape sh) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  const int token_bytes = sh.bn * 128;
  const SmallBars bars(smem, sh.stages);
  uint8_t* pipe = smem + 1024;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t m0 = (int64_t)blockIdx.y * sh.bn;
  // this CTA's rows of the vocabulary, in units of 32
  const int64_t units = (p.N + 31) / 32;
  const int64_t u0 = units * blockIdx.x / gridDim.x, u1 = units * (blockIdx.x + 1) / gridDim.x;
  const int tiles = (int)((u1 - u0 + 3) / 4);
  const int iters = (int)((p.K + 63) / 64);
  const uint32_t acc_stride = small_tmem_cols(sh.bn), tmem_cols = 2 * acc_stride;
  small_setup(bars, sh.stages, tmem_cols, kWarps);
  const uint32_t tmem_base = *bars.tmem_slot;
  grid_dependency_wait();

  if (warp == 0) {
    int stage = 0;
    uint32_t phase = 0;
    bool ok = true;
    const uint32_t base = smem_u32(pipe);
    for (int t = 0; t < tiles && ok; ++t) {
      const int64_t first = u0 + 4 * t;
      const int n_units = u1 - first < 4 ? (int)(u1 - first) : 4;
      for (int it = 0; it < iters; ++it) {
        ok = __all_sync(0xffffffffu, mbar_wait(&bars.empty[stage], phase ^ 1u, bars.abort_flag));
        if (!ok) {
          if (lane == 0) report(p.status, bars.abort_flag, METIS_DEV_TIMEOUT_MMA);
          break;
        }
        if (elect_one()) {
          const uint32_t st = base + stage * sh.stage_bytes, sw = st + token_bytes, bar = smem_u32(&bars.full[stage]);
          mbar_expect_tx_addr(bar, (uint32_t)(token_bytes + n_units * 4096));
          for (int u = 0; u < n_units; ++u) tma_load_2d_addr(sw + u * 4096, &map_w, it * 64, (int32_t)(first + u) * 32, bar);
          tma_load_2d_addr(st, &map_t, it * 64, (int32_t)m0, bar);
        }
        if (++stage == sh.stages) { stage = 0; phase ^= 1u; }
      }
    }
    grid_launch_dependents();
  } else if (warp == 1) {
    int stage = 0;
    uint32_t phase = 0;
    bool ok = true, issued = false;
    const uint32_t base = smem_u32(pipe), idesc = idesc_bf16(sh.bn);
    for (int t = 0; t < tiles && ok; ++t) {
      const int buf = t & 1;
      if (t > 1) {
        ok = __all_sync(0xffffffffu, mbar_wait(&bars.acc_empty[buf], (uint32_t)((t >> 1) - 1) & 1u, bars.abort_flag));
        if (!ok) {
          if (lane == 0) report(p.status, bars.abort_flag, METIS_DEV_TIMEOUT_EPI);
          break;
        }
      }
      tc_fence_after();
      for (int it = 0; it < iters; ++it) {
        ok = __all_sync(0xffffffffu, mbar_wait(&bars.full[stage], phase, bars.abort_flag));
        if (!ok) {
          if (lane == 0) report(p.status, bars.abort_flag, METIS_DEV_TIMEOUT_TMA);
          break;
        }
        tc_fence_after();
        if (elect_one()) {
          const uint32_t st = base + stage * sh.stage_bytes;
          small_mma<false>(tmem_base + buf * acc_stride, st + token_bytes, st, idesc, it == 0);
          tc_commit(&bars.empty[stage]);
          if (it == iters - 1) tc_commit(&bars.acc_full[buf]);
        }
        issued = true;
        if (++stage == sh.stages) { stage = 0; phase ^= 1u; }
      }
    }
    if (!ok && issued && elect_one()) {
      tc_commit(bars.drain);
      const uint64_t t0 = global_ns();
      while (!mbar_try(bars.drain, 0) && global_ns() - t0 < kWaitLimitNs) {}
    }
    __syncwarp();
  } else {
    const int q = warp & 3;
    const int c0 = ((warp - 2) >> 2) * 32;                 // this warp's first token of the tile
    const int64_t token = m0 + c0 + lane;                  // lane l looks after the target of token l
    int64_t target = -1;
    if (token < p.M && c0 < sh.bn) {
      const int64_t t = p.target[token];
      if (t != p.ignore && t >= 0 && t < p.vocab) target = t;
    }
    float m[32], s[32], e[32];
#pragma unroll
    for (int i = 0; i < 32; ++i) { m[i] = kNoLogit; s[i] = 0.0f; e[i] = 0.0f; }
    for (int t = 0; t < tiles; ++t) {
      const int buf = t & 1;
      const int64_t first = u0 + 4 * t, row = first * 32 + q * 32 + lane;
      if (!mbar_wait(&bars.acc_full[buf], (uint32_t)(t >> 1) & 1u, bars.abort_flag)) {
        if (lane == 0) report(p.status, bars.abort_flag, METIS_DEV_TIMEOUT_MMA);
        break;
      }
      tc_fence_after();
      uint32_t r[32];
      tc_load32(tmem_base + ((uint32_t)(q * 32) << 16) + buf * acc_stride + c0, r);
      tc_wait_ld(r);
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive_addr(smem_u32(&bars.acc_empty[buf]));
      // targets among these 32 rows, seldom any: left out (head_rows_kernel adds them)
      uint32_t hits = __ballot_sync(0xffffffffu, first + q < u1 && (target >> 5) == first + q);
      while (hits) {
        const int who = __ffs(hits) - 1;
        hits &= hits - 1;
        const bool at = (int)(__shfl_sync(0xffffffffu, target, who) & 31) == lane;
#pragma unroll
        for (int i = 0; i < 32; ++i) if (i == who && at) r[i] = kMinusInfinity;
      }
      if (first + q < u1 && row < p.N) {
#pragma unroll
        for (int i = 0; i < 32; ++i) stats_add<kEntropy>(__uint_as_float(r[i]) * p.scale_log2e, m[i], s[i], e[i]);
      }
    }
    // lanes into one: after five steps lane l has the statistics of token l, half of the tokens leaving at each
    RowStats a[32];
#pragma unroll
    for (int i = 0; i < 32; ++i) a[i] = RowStats{s[i] == 0.0f ? -INFINITY : m[i], m[i] == INFINITY ? NAN : s[i], e[i]};
#pragma unroll
    for (int off = 16; off >= 1; off >>= 1) {
      const bool upper = (lane & off) != 0;
#pragma unroll
      for (int j = 0; j < off; ++j) {
        RowStats send = upper ? a[j] : a[j + off], keep = upper ? a[j + off] : a[j];
        send.m = __shfl_xor_sync(0xffffffffu, send.m, off);
        send.s = __shfl_xor_sync(0xffffffffu, send.s, off);
        if constexpr (kEntropy) send.e = __shfl_xor_sync(0xffffffffu, send.e, off);
        stats_merge<kEntropy>(keep, send);
        a[j] = keep;
      }
    }
    if (token < p.M && c0 < sh.bn) {
      const int64_t slot = ((int64_t)blockIdx.x * 4 + q) * p.stats_ld + token;
      p.stats[slot] = make_float2(a[0].m, a[0].s);
      if constexpr (kEntropy) p.stats_e[slot] = a[0].e;
    }
  }
  tc_fence_before();
  __syncthreads();
  small_free(tmem_base, tmem_cols);
}

// ---- host side ------------------------------------------------------------------------------------------------

// Clusters of `splits` CTAs with `smem` bytes each that run at once on the current device, asked once.
static int resident_clusters(int splits, int which, const void* kern, int smem) {
  static std::atomic<int> known[64][9][2][2];
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 1;
  std::atomic<int>& slot = known[dev][splits][which & 1][which >> 1];
  int n = slot.load(std::memory_order_relaxed);
  if (n == 0) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)splits);
    cfg.blockDim = dim3(kSmallThreads);
    cfg.dynamicSmemBytes = (size_t)smem;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = (unsigned)splits;
    attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmallBudgetAlone) != cudaSuccess ||
        cudaOccupancyMaxActiveClusters(&n, kern, &cfg) != cudaSuccess || n < 1) {
      cudaGetLastError();
      n = 1;
    }
    slot.store(n, std::memory_order_relaxed);
  }
  return n;
}

// Shape of a product, and its time in us by the model that chooses it.  A block's two copies take an SM 0.23 us at least, however small; its
// bytes come at 108 GB/s an SM and 10 TB/s over all of them, the weight from memory at 5.5 TB/s.  Around that 4.2 us, 13 ns for each token of a
// tile and 0.15 ns for each element (drain and epilogue), 1.5 us and 10 ns a token more where a cluster meets, and 4 us for every further
// round of CTAs.  Measured, us, by rows of a tile, blocks to a stage, splits: 1 x 3584 x 18944 26.4 (128, 2, 4), 27.8 (64, 4, 4), 35 (128, 1, 3),
// 47 (32, 4, 1); 64 x 3584 x 18944 30.1 (128, 2, 4), 34.0 (128, 1, 5); 256 x 3584 x 3584 21.1 (128, 1, 4), 30.2 (32, 1, 1); 256 x 1536 x 1536
// 14.0 (64, 1, 4), 16.2 (64, 1, 2); 1 x 18944 x 3584 24.5 (128, 2, 1), 25.3 (64, 4, 1).
SmallPlan plan_dense_small(int64_t M, int64_t N, int64_t K, bool w_mn) {
  SmallPlan best = {};
  float best_rank = 1e30f;
  const int64_t blocks = ceil_div(K, 64), sms = device_sm_count();
  const int64_t token_tiles = ceil_div(M, 256);
  const int bn = (int)(ceil_div(ceil_div(M, token_tiles), 16) * 16);
  const void* kern = w_mn ? reinterpret_cast<const void*>(dense_small_kernel<true>) : reinterpret_cast<const void*>(dense_small_kernel<false>);
  const float memory_us = (float)(2 * N * K) / 5.5e6f;
  for (int alone = 1; alone >= 0; --alone) {               // (deeper pipelines first, where the model sees no difference)
    const int budget = alone ? kSmallBudgetAlone : kSmallBudget;
    for (int rows = 128; rows >= (w_mn ? 64 : 32); rows >>= 1) {
      const int block_bytes = (rows + bn) * 128;
      int kb = 4;                                          // a stage of up to 48 KiB, four of them at least
      while (kb > 1 && (kb * block_bytes > 48 * 1024 || 4 * kb * block_bytes > budget - 2048 - (128 - rows) * 128)) kb >>= 1;
      const int stage_bytes = kb * block_bytes;
      int stages = (budget - 2048 - (128 - rows) * 128) / stage_bytes;
      if (stages > 24) stages = 24;
      if (stages < 3 || 2048 + bn * 512 > budget) continue;
      for (int splits = 1; splits <= 8; ++splits) {
        const int64_t per = ceil_div(blocks, splits);
        if (splits > 1 && (per < 4 || ceil_div(blocks, per) != splits)) continue;
        const int64_t clusters = ceil_div(N, rows) * token_tiles, at_once = resident_clusters(splits, alone + 2 * w_mn, kern, budget);
        const int64_t rounds = ceil_div(clusters, at_once), ctas = (clusters < at_once ? clusters : at_once) * splits;
        const float sharing = ctas > sms ? (float)ctas / (float)sms : 1.0f;
        float block_us = sharing * (float)block_bytes / 108e3f;
        const float all_us = (float)block_bytes * (float)ctas / 10e6f, trip_us = 0.23f;
        if (block_us < all_us) block_us = all_us;
        if (block_us < trip_us) block_us = trip_us;
        const float feed_us = (float)(rounds * per) * block_us;
        const float rest = 4.0f * (float)(rounds - 1) + 4.2f + 0.013f * (float)bn + 0.00015f * (float)(rows * bn) + (splits > 1 ? 1.5f + 0.01f * (float)bn : 0.0f);
        const bool bound = feed_us < memory_us;            // by memory: of such shapes the one that feeds faster
        const float us = (bound ? memory_us : feed_us) + rest, rank = us + 0.3f * (bound ? feed_us : memory_us);
        if (rank < best_rank) {
          best_rank = rank;
          best.us = us;
          best.sh = SmallShape{rows, bn, kb, stages, stage_bytes, splits, (int)per};
        }
      }
    }
  }
#ifdef METIS_TIMING_KNOBS
  if (const char* e = getenv("METIS_DEV_SMALL_SHAPE")) {       // rows,kb,splits,alone
    int r, kb, sp, al;
    if (sscanf(e, "%d,%d,%d,%d", &r, &kb, &sp, &al) == 4) {
      const int stage_bytes = kb * (r + bn) * 128;
      int stages = ((al ? kSmallBudgetAlone : kSmallBudget) - 2048 - (128 - r) * 128) / stage_bytes;
      if (stages > 24) stages = 24;
      const int64_t per = ceil_div(blocks, sp);
      if (stages >= 2 && ceil_div(blocks, per) == sp) best.sh = SmallShape{r, bn, kb, stages, stage_bytes, sp, (int)per};
    }
  }
#endif
  return best;
}

// d = epilogue(T W^T) for tokens t [M, K] and a weight w [N, K] (or [K, N])
int32_t launch_dense_small(const SmallShape& sh, const void* t, int64_t ldt, const void* w, bool w_mn, int64_t ldw, const DenseParams& p, cudaStream_t st) {
  const CUtensorMapDataType dt = CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  CUtensorMap mt, mw;
  if (int32_t rc = make_map(&mt, dt, 2, t, p.K, p.M, ldt * 2, 64, sh.bn, "tokens")) return rc;
  if (w_mn) { if (int32_t rc = make_map(&mw, dt, 2, w, p.N, p.K, ldw * 2, 64, 64, "weight (MN-major)")) return rc; }
  else      { if (int32_t rc = make_map(&mw, dt, 2, w, p.K, p.N, ldw * 2, 64, sh.rows, "weight (K-major)")) return rc; }
  const int pipe = sh.stages * sh.stage_bytes + (128 - sh.rows) * 128, sums = sh.bn * 512;
  const int smem = 2048 + (pipe > sums ? pipe : sums);
  auto kern = w_mn ? dense_small_kernel<true> : dense_small_kernel<false>;
  static std::atomic<uint64_t> done[2];
  METIS_CUDA_OK(allow_shared(reinterpret_cast<const void*>(kern), kSmallBudgetAlone, done[w_mn]));
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(ceil_div(p.N, sh.rows) * sh.splits), (unsigned)ceil_div(p.M, sh.bn), 1);
  cfg.blockDim = dim3(kSmallThreads, 1, 1);
  cfg.dynamicSmemBytes = (size_t)smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = launch_overlap_enabled(kLaunchGemm) ? 1 : 0;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = (unsigned)sh.splits;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  METIS_CUDA_OK(cudaLaunchKernelEx(&cfg, kern, mw, mt, p, sh));
  dense_launches.fetch_add(1, std::memory_order_relaxed);
  return METIS_OK;
}

int64_t small_stats_slots(int64_t V) {
  const int64_t units = ceil_div(V, 32), sms = device_sm_count();
  return 4 * (units < sms ? units : sms);
}

// p.stats and p.stats_e of up to 64 tokens h [M, K] against a vocabulary w [V, K]: small_stats_slots(V) slots
int32_t launch_dense_small_stats(const void* h, int64_t ldh, const void* w, int64_t ldw, const DenseParams& p, cudaStream_t st) {
  SmallShape sh = {};
  sh.rows = 128;
  sh.bn = (int)(ceil_div(p.M, 16) * 16);
  sh.stage_bytes = (sh.rows + sh.bn) * 128;
  sh.stages = kStatsBudget / sh.stage_bytes;
  const CUtensorMapDataType dt = CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  CUtensorMap mt, mw;
  if (int32_t rc = make_map(&mt, dt, 2, h, p.K, p.M, ldh * 2, 64, sh.bn, "h")) return rc;
  if (int32_t rc = make_map(&mw, dt, 2, w, p.K, p.N, ldw * 2, 64, 32, "w")) return rc;
  const int smem = 2048 + sh.stages * sh.stage_bytes;
  const bool wide = sh.bn > 32;
  auto kern = p.stats_e ? (wide ? dense_small_stats_kernel<true, 8> : dense_small_stats_kernel<true, 4>)
                        : (wide ? dense_small_stats_kernel<false, 8> : dense_small_stats_kernel<false, 4>);
  static std::atomic<uint64_t> done[4];
  METIS_CUDA_OK(allow_shared(reinterpret_cast<const void*>(kern), 2048 + kStatsBudget, done[2 * wide + (p.stats_e != nullptr)]));
  METIS_CUDA_OK(launch_counted(kLaunchGemm, kern, dim3((unsigned)(small_stats_slots(p.N) / 4)), dim3(wide ? 320 : 192), (size_t)smem, st, mw, mt, p, sh));
  return METIS_OK;
}

}  // namespace metis
