// bf16 products on CTA pairs (tcgen05 kind::f16, cta_group::2) with the epilogues of the layers that stay in bf16, for sm_100a:
//
//   D [M, N] = A B^T, A [M, K] and B [N, K], either operand stored with the contraction in its rows instead (MN-major: the
//   gradients read their operands as they lie, nothing is transposed in memory), and behind it
//     linear   act(D + bias) * gate + residual in bf16, and the value in front of act where a backward pass will want it
//     stats    for each row the maximum of the logits and the sum of their exponentials over this tile's columns, and the entropy's
//              sum, all without the target's: the logits themselves are never stored
//     grad     the logits' gradient (softmax - one-hot) times the row's weight, in bf16: the operand of the two products behind it
//     sum      D, or D plus an fp32 addend, in bf16 or fp32: gradients, summed over pieces of the vocabulary
//
// A pair computes 256 x 256 tiles: CTA r has rows [128 r, +128) of A and of B and rows [128 r, +128) of the accumulator.  Two whole
// accumulators fit tensor memory (2 x 256 columns), so the epilogue of a tile runs beside all of the next tile's MMAs.  A stage is 64
// elements of the contraction (32 KiB per CTA), six of them are in flight.  Roles as in the NVFP4 product: warp 0 loads, warp 1 of
// the leader issues, warps 2 to 9 are the epilogue (two for each 32-lane quarter of tensor memory, 128 columns each).
// No copy is multicast.  Every wait is bounded; both CTAs meet at a cluster barrier before they free tensor memory.
#include "dense.cuh"
#include "pair.cuh"

namespace metis {

std::atomic<int64_t> dense_launches{0};

enum DenseEpilogue { kEpiLinear, kEpiLinearWide, kEpiLinearOdd, kEpiStats, kEpiStatsEntropy, kEpiGrad, kEpiSum, kEpiSumF32 };

template <int kEpi> struct DenseCfg {
  static constexpr bool kOperands = kEpi == kEpiLinearWide || kEpi == kEpiLinearOdd;
  static constexpr int kParts = 2;                         // epilogue warps for each 32-lane quarter of tensor memory
  static constexpr int kStages = kOperands ? 5 : 6;
  static constexpr int kHalfBytes = 128 * 128;             // 128 rows x 64 elements of A or of B
  static constexpr int kBoxBytes = 64 * 128;               // one MN-major box: 64 contraction rows x 64 elements
  static constexpr int kStageBytes = 2 * kHalfBytes;
  static constexpr int kEpilogueWarps = 4 * kParts;
  static constexpr int kChunks = 8 / kParts;               // of 32 columns, that a warp takes of a tile
  static constexpr int kThreads = 64 + 32 * kEpilogueWarps;
  // for each epilogue warp: buffers of 32 rows x 64 bytes for what is stored, then two for the pieces of the operands
  static constexpr int kStores = kEpi == kEpiLinearOdd ? 1 : 2;
  static constexpr int kPieceBytes = kEpi == kEpiLinearOdd ? 32 * 80 : 2048;
  static constexpr int kWarpBytes = kStores * 2048 + (kOperands ? 2 * kPieceBytes : 0);
  static constexpr int kStagingBytes = kEpilogueWarps * kWarpBytes;
  static constexpr int kSmemBytes = kStages * kStageBytes + kStagingBytes + 1024 + 256;
};
static_assert(DenseCfg<kEpiLinearOdd>::kWarpBytes % 512 == 0, "the swizzle of a stored piece counts from 512 bytes");
static_assert(DenseCfg<kEpiLinear>::kSmemBytes <= 227 * 1024 && DenseCfg<kEpiLinearWide>::kSmemBytes <= 227 * 1024 && DenseCfg<kEpiLinearOdd>::kSmemBytes <= 227 * 1024);

// ---- epilogue pieces ----------------------------------------------------------------------------------------

// A warp's buffers of 32 rows x 64 bytes, used in turn by the stores that leave through the TMA unit.
struct Staging {
  uint8_t* base;
  uint32_t flip = 0;
  __device__ __forceinline__ uint8_t* next() {             // (the stores of one buffer are read while the other is filled)
    uint8_t* buf = base + flip * 2048;
    flip ^= 1u;
    if ((threadIdx.x & 31) == 0) bulk_store_wait_read<1>();
    __syncwarp();
    return buf;
  }
  // one for other uses: no store reads it any more, and no lane
  __device__ __forceinline__ uint8_t* idle() {
    if ((threadIdx.x & 31) == 0) bulk_store_wait_read<0>();
    __syncwarp();
    return base;
  }
};

// Two such pieces of two tensors at once: one wait for the buffers, one fence.
__device__ __forceinline__ void store_two_tma(Staging& st, const CUtensorMap* map0, const uint32_t (&w0)[16], const CUtensorMap* map1, const uint32_t (&w1)[16],
                                              int32_t x, int32_t row0) {
  const int lane = threadIdx.x & 31, swz = (lane >> 1) & 3;
  uint8_t* buf = st.idle();
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    *reinterpret_cast<uint4*>(buf + lane * 64 + ((k ^ swz) << 4)) = make_uint4(w0[4 * k], w0[4 * k + 1], w0[4 * k + 2], w0[4 * k + 3]);
    *reinterpret_cast<uint4*>(buf + 2048 + lane * 64 + ((k ^ swz) << 4)) = make_uint4(w1[4 * k], w1[4 * k + 1], w1[4 * k + 2], w1[4 * k + 3]);
  }
  fence_async_shared();
  __syncwarp();
  if (lane == 0) {
    tma_store_2d(map0, smem_u32(buf), x, row0);
    tma_store_2d(map1, smem_u32(buf) + 2048, x, row0);
  }
}

// Three, the third in a buffer of the caller's.
__device__ __forceinline__ void store_three_tma(Staging& st, uint8_t* third, const CUtensorMap* map0, const uint32_t (&w0)[16], const CUtensorMap* map1,
                                                const uint32_t (&w1)[16], const CUtensorMap* map2, const uint32_t (&w2)[16], int32_t x, int32_t row0) {
  const int lane = threadIdx.x & 31, swz = (lane >> 1) & 3;
  uint8_t* buf = st.idle();
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const int at = lane * 64 + ((k ^ swz) << 4);
    *reinterpret_cast<uint4*>(buf + at) = make_uint4(w0[4 * k], w0[4 * k + 1], w0[4 * k + 2], w0[4 * k + 3]);
    *reinterpret_cast<uint4*>(buf + 2048 + at) = make_uint4(w1[4 * k], w1[4 * k + 1], w1[4 * k + 2], w1[4 * k + 3]);
    *reinterpret_cast<uint4*>(third + at) = make_uint4(w2[4 * k], w2[4 * k + 1], w2[4 * k + 2], w2[4 * k + 3]);
  }
  fence_async_shared();
  __syncwarp();
  if (lane == 0) {
    tma_store_2d(map0, smem_u32(buf), x, row0);
    tma_store_2d(map1, smem_u32(buf) + 2048, x, row0);
    tma_store_2d(map2, smem_u32(third), x, row0);
  }
}

// 32 rows x 64 bytes, one row per lane (four 16-byte pieces), through shared memory to the tensor at (row0, x): 64-byte swizzle.
template <int kStores = 2>
__device__ __forceinline__ void store_piece_tma(Staging& st, const CUtensorMap* map, const uint32_t (&w)[16], int32_t x, int32_t row0) {
  const int lane = threadIdx.x & 31, swz = (lane >> 1) & 3;
  uint8_t* buf = kStores == 2 ? st.next() : st.idle();
#pragma unroll
  for (int k = 0; k < 4; ++k)
    *reinterpret_cast<uint4*>(buf + lane * 64 + ((k ^ swz) << 4)) = make_uint4(w[4 * k], w[4 * k + 1], w[4 * k + 2], w[4 * k + 3]);
  fence_async_shared();
  __syncwarp();
  if (lane == 0) tma_store_2d(map, smem_u32(buf), x, row0);
}

// The same 32 x 32 bf16 for rows that no TMA store reaches (a pitch or an address that 16 bytes do not divide): a row at a time,
// 64 contiguous bytes of it by the 32 lanes.  (Two rows at a time by words of two elements, shifted where a row begins in the middle of
// one: 8192 x 8961 x 1536 340 us in place of 180.)
__device__ __forceinline__ void store_piece_rows(Staging& st, __nv_bfloat16* out, int64_t ld, const uint32_t (&w)[16], int64_t col0, int64_t row0,
                                                 int64_t M, int64_t N) {
  const int lane = threadIdx.x & 31, swz = (lane >> 1) & 3;
  uint8_t* buf = st.idle();
#pragma unroll
  for (int k = 0; k < 4; ++k)
    *reinterpret_cast<uint4*>(buf + lane * 64 + ((k ^ swz) << 4)) = make_uint4(w[4 * k], w[4 * k + 1], w[4 * k + 2], w[4 * k + 3]);
  __syncwarp();
  const bool live = col0 + lane < N;
  unsigned short* to = reinterpret_cast<unsigned short*>(out) + row0 * ld + col0 + lane;
#pragma unroll
  for (int r0 = 0; r0 < 32; r0 += 8) {                     // eight rows on their way at a time
    unsigned short v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int r = r0 + i;
      v[i] = *reinterpret_cast<const unsigned short*>(buf + r * 64 + (((lane >> 3) ^ ((r >> 1) & 3)) << 4) + (lane & 7) * 2);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) if (live && row0 + r0 + i < M) to[(r0 + i) * ld] = v[i];
  }
  __syncwarp();
}

// This lane's 32 elements of a row of a bf16 operand of the epilogue, as words, where no TMA load reads it (a pitch or an address that 16
// bytes do not divide): the warp reads row after row, a lane an element, eight rows in flight, and turns them through shared memory.
// What lies outside the tensor is zero.
__device__ __forceinline__ void load_piece_rows(Staging& st, const __nv_bfloat16* src, int64_t ld, int64_t col0, int64_t row0, int64_t M, int64_t N,
                                                uint32_t (&w)[16]) {
  const int lane = threadIdx.x & 31, swz = (lane >> 1) & 3;
  uint8_t* buf = st.idle();
  const unsigned short* s = reinterpret_cast<const unsigned short*>(src) + row0 * ld + col0 + lane;
  const bool live = col0 + lane < N;
  for (int r0 = 0; r0 < 32; r0 += 8) {
    unsigned short v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = live && row0 + r0 + i < M ? s[(r0 + i) * ld] : (unsigned short)0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int r = r0 + i;
      *reinterpret_cast<unsigned short*>(buf + r * 64 + (((lane >> 3) ^ ((r >> 1) & 3)) << 4) + (lane & 7) * 2) = v[i];
    }
  }
  __syncwarp();
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const uint4 q = *reinterpret_cast<const uint4*>(buf + lane * 64 + ((k ^ swz) << 4));
    w[4 * k] = q.x; w[4 * k + 1] = q.y; w[4 * k + 2] = q.z; w[4 * k + 3] = q.w;
  }
  __syncwarp();
}

__device__ __forceinline__ void add_bias32(float (&v)[32], const DenseParams& p, int64_t col0, bool full) {
  if (p.bias_f32) {
    const float* b = static_cast<const float*>(p.bias) + col0;
#pragma unroll
    for (int i = 0; i < 32; ++i) if (full || col0 + i < p.N) v[i] += b[i];
  } else {
    const __nv_bfloat16* b = static_cast<const __nv_bfloat16*>(p.bias) + col0;
#pragma unroll
    for (int i = 0; i < 32; ++i) if (full || col0 + i < p.N) v[i] += __bfloat162float(b[i]);
  }
}

// An operand of the epilogue, [M, N] bf16.  Its pieces of 32 rows x 64 bytes come into a buffer of the warp's by asynchronous copies, the
// next one on its way while the last one is worked on; each fetch is a group of copies, empty or not.
//   rows of whole 16-byte pieces: four lanes a row, so that a copy takes whole sectors; the ragged end of a row is load_piece_rows'
//   any others (kOdd): the aligned 16 bytes that hold them, five a row since a row may begin anywhere in them, shifted when they are taken (what
//     lies beside the piece in them belongs to the same allocation and is not used).  Without it every piece waits for four rounds of
//     loads: 8192 x 8961 x 1536 with silu, gate and residual 840 us, by 4-byte copies 574, 8960 columns 199.
template <bool kOdd> struct EpilogueOperand {
  const __nv_bfloat16* src;                                // null: there is none
  int64_t ld;
  bool wide;                                               // 16-byte aligned rows
  uint8_t* buf;
  __device__ __forceinline__ void fetch(bool valid, int64_t col0, int64_t row0, int64_t M, int64_t N) {
    __syncwarp();                                          // every lane has read what the buffer held
    const int lane = threadIdx.x & 31;
    const uint32_t to = smem_u32(buf);
    if constexpr (kOdd) {
      if (src && valid) {
        const int bytes = N - col0 < 32 ? 2 * (int)(N - col0) : 64, rows = M - row0 < 32 ? (int)(M - row0) : 32;
#pragma unroll
        for (int i = 0; i < 5; ++i) {
          const int at = i * 32 + lane, r = at / 5, k = at - r * 5;
          const uintptr_t first = reinterpret_cast<uintptr_t>(src + (row0 + r) * ld + col0);
          if (r < rows && 16 * k < bytes + (int)(first & 15))
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to + at * 16), "l"((first & ~(uintptr_t)15) + 16 * k) : "memory");
        }
      }
    } else {
      if (src && wide && valid && col0 + 32 <= N) {
        const __nv_bfloat16* at = src + (row0 + (lane >> 2)) * ld + col0 + (lane & 3) * 8;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int r = 8 * i + (lane >> 2);
          if (row0 + r < M)
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to + r * 64 + (((lane & 3) ^ ((r >> 1) & 3)) << 4)), "l"(at + 8 * i * ld) : "memory");
        }
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  }
  // this lane's 32 elements of its row, of the piece that was fetched two groups ago, or in the last group
  __device__ __forceinline__ void take(uint32_t (&w)[16], int64_t col0, int64_t row0, bool last) {
    const int lane = threadIdx.x & 31;
    if (last) asm volatile("cp.async.wait_group 0;" ::: "memory");
    else asm volatile("cp.async.wait_group 1;" ::: "memory");
    __syncwarp();
    if constexpr (kOdd) {
      const uint32_t off = (uint32_t)(reinterpret_cast<uintptr_t>(src + (row0 + lane) * ld + col0) & 15);
      uint32_t x[20];
#pragma unroll
      for (int k = 0; k < 5; ++k) {
        const uint4 t = *reinterpret_cast<const uint4*>(buf + lane * 80 + 16 * k);
        x[4 * k] = t.x; x[4 * k + 1] = t.y; x[4 * k + 2] = t.z; x[4 * k + 3] = t.w;
      }
#pragma unroll
      for (int k = 0; k < 18; ++k) x[k] = (off & 8) ? x[k + 2] : x[k];
#pragma unroll
      for (int k = 0; k < 17; ++k) x[k] = (off & 4) ? x[k + 1] : x[k];
#pragma unroll
      for (int k = 0; k < 16; ++k) w[k] = __funnelshift_r(x[k], x[k + 1], (off & 2) * 8);
    } else {
      const int swz = (lane >> 1) & 3;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const uint4 t = *reinterpret_cast<const uint4*>(buf + lane * 64 + ((k ^ swz) << 4));
        w[4 * k] = t.x; w[4 * k + 1] = t.y; w[4 * k + 2] = t.z; w[4 * k + 3] = t.w;
      }
    }
  }
};

// The output alone: bias and activation, a store through the TMA unit.
__device__ __forceinline__ void linear_chunk(const DenseParams& p, Staging& st, const CUtensorMap* map_d, const uint32_t (&r)[32], int64_t row0, int64_t col0) {
  float v[32];
#pragma unroll
  for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(r[i]);
  if (p.bias) add_bias32(v, p, col0, col0 + 32 <= p.N);
  activate_all(p.act, v);
  uint32_t w[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) w[i] = pack_bf16(v[2 * i], v[2 * i + 1]);
  if (p.d_wide) store_piece_tma(st, map_d, w, (int32_t)col0, (int32_t)row0);
  else store_piece_rows(st, p.d, p.ldd, w, col0, row0, p.M, p.N);
}

// With gate, residual, or what the gradients need: several tensors of the output's size pass by, and each adds its time to the layer's
// (the tensor pipe is busy 0.59 of the time with four of them, 0.95 with the output alone).  What is read comes by asynchronous copies of the
// load/store unit a piece ahead; what is written leaves by the TMA unit, all of it behind one fence where there are buffers for it (without
// a residual its buffer is the third).  8192 x 8960 x 1536, us: plain 152, silu with slopes 184, silu and gate 200, and slopes and act(z)
// 224 (240 warm; 270 with a wait and a fence for the output alone), gate and residual 192, all of them 248 (272 warm); five
// stages in place of six, for the buffers' sake, cost a plain layer 4.  It is a warp's chain that takes the time, not the bytes: one row of
// the gate for all takes as long.  Tried with two outputs (silu, gate, one tensor for the gradients / gate and residual, 204 / 187 by this
// form): loads into registers where they are used 238 / 220; loads by the TMA unit, which queue behind the tiles' own, 209 / -; 16 warps of 96
// registers 258 / 269, with four stages 275 / 236; stores by the load/store unit 235 / 188.  `next`: the piece that this warp takes after this one.
struct PieceAt {
  bool valid;
  int64_t row0, col0;
};
template <bool kOdd>
__device__ __forceinline__ void linear_wide_chunk(const DenseParams& p, Staging& st, const CUtensorMap* map_d, const CUtensorMap* map_s, const CUtensorMap* map_a, EpilogueOperand<kOdd>& gate,
                                                  EpilogueOperand<kOdd>& residual, const uint32_t (&r)[32], int64_t row0, int64_t col0, const PieceAt& next) {
  constexpr int kStores = kOdd ? 1 : 2;
  const bool full = col0 + 32 <= p.N;
  float v[32];
#pragma unroll
  for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(r[i]);
  uint32_t w[16], slopes[16], act[16];
  if (p.bias) add_bias32(v, p, col0, full);
  if (p.slope) activate_both_all(p.act, v, slopes);
  else activate_all(p.act, v);
  if (p.act_out) {
#pragma unroll
    for (int i = 0; i < 16; ++i) act[i] = pack_bf16(v[2 * i], v[2 * i + 1]);
  }
  // the stores' fence waits for copies on their way as well: with three outputs they start behind it (silu, gate, slopes and act(z) 228 -> 224
  // us, 250 -> 240 warm), without they are wanted early (gate and residual 188, behind it 192)
  const bool late = p.slope && p.act_out;
  const bool together = !kOdd && p.d_wide && !(p.slope && p.act_out && residual.src);
  if (!together) {
    if (p.slope) store_piece_tma<kStores>(st, map_s, slopes, (int32_t)col0, (int32_t)row0);
    if (p.act_out) store_piece_tma<kStores>(st, map_a, act, (int32_t)col0, (int32_t)row0);
  }
  if (gate.src) {
    if (kOdd || (gate.wide && full)) gate.take(w, col0, row0, false);
    else load_piece_rows(st, gate.src, gate.ld, col0, row0, p.M, p.N, w);
#pragma unroll
    for (int i = 0; i < 16; ++i) { v[2 * i] *= bf16_lo(w[i]); v[2 * i + 1] *= bf16_hi(w[i]); }
  }
  if (!late) gate.fetch(next.valid, next.col0, next.row0, p.M, p.N);
  if (residual.src) {
    if (kOdd || (residual.wide && full)) residual.take(w, col0, row0, late);        // (late: no group of the gate lies behind it)
    else load_piece_rows(st, residual.src, residual.ld, col0, row0, p.M, p.N, w);
#pragma unroll
    for (int i = 0; i < 16; ++i) { v[2 * i] += bf16_lo(w[i]); v[2 * i + 1] += bf16_hi(w[i]); }
  }
  if (!late) residual.fetch(next.valid, next.col0, next.row0, p.M, p.N);
#pragma unroll
  for (int i = 0; i < 16; ++i) w[i] = pack_bf16(v[2 * i], v[2 * i + 1]);
  if (together && p.slope && p.act_out) store_three_tma(st, residual.buf, map_s, slopes, map_a, act, map_d, w, (int32_t)col0, (int32_t)row0);
  else if (together && p.slope) store_two_tma(st, map_s, slopes, map_d, w, (int32_t)col0, (int32_t)row0);
  else if (together && p.act_out) store_two_tma(st, map_a, act, map_d, w, (int32_t)col0, (int32_t)row0);
  else if (p.d_wide) store_piece_tma<kStores>(st, map_d, w, (int32_t)col0, (int32_t)row0);
  else store_piece_rows(st, p.d, p.ldd, w, col0, row0, p.M, p.N);
  if (late) {
    gate.fetch(next.valid, next.col0, next.row0, p.M, p.N);
    residual.fetch(next.valid, next.col0, next.row0, p.M, p.N);
  }
}

// The statistics of this lane's row take 32 more logits: maximum of the chunk, then one exponential per element.
template <bool kEntropy>
__device__ __forceinline__ void stats_chunk(const DenseParams& p, RowStats& a, const uint32_t (&r)[32], int64_t col0) {
  float v[32];
#pragma unroll
  for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(r[i]) * p.scale_log2e;
  const bool full = col0 + 32 <= p.N;
  float m = a.m;
  if (full) {
#pragma unroll
    for (int i = 0; i < 32; i += 2) m = max3(m, v[i], v[i + 1]);
  } else {
#pragma unroll
    for (int i = 0; i < 32; ++i) if (col0 + i < p.N) m = fmaxf(m, v[i]);
  }
  const float base = stats_base(m);
  const float f = exp2_fast(a.m - base);
  float s[2] = {0.0f, 0.0f}, e[2] = {0.0f, 0.0f};
#pragma unroll
  for (int i = 0; i < 32; ++i) {
    if (full || col0 + i < p.N) {
      const float d = v[i] - base;
      const float x = exp2_fast(d);
      s[i & 1] += x;
      if constexpr (kEntropy) e[i & 1] = fmaf(x, fmaxf(d, -1e30f), e[i & 1]);     // (a logit of -infinity adds 0)
    }
  }
  if constexpr (kEntropy) {
    const float d = a.m == -INFINITY ? 0.0f : a.m - base;
    a.e = fmaf(f, fmaf(d, a.s, a.e), e[0] + e[1]);
  }
  a.s = fmaf(a.s, f, s[0] + s[1]);
  a.m = m;
}

// ---- the kernel ---------------------------------------------------------------------------------------------

template <bool kAMn, bool kBMn, int kEpi>
__global__ void __launch_bounds__(DenseCfg<kEpi>::kThreads, 1)
dense_gemm_pair_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b, const __grid_constant__ CUtensorMap map_d,
                       const __grid_constant__ CUtensorMap map_s, const __grid_constant__ CUtensorMap map_act, const DenseParams p) {
  using Cfg = DenseCfg<kEpi>;
  constexpr int kStages = Cfg::kStages;
  constexpr int BN = 256;

  extern __shared__ uint8_t smem_raw[];
  // the dynamic window starts at the same offset in both CTAs: descriptors and barrier offsets are valid across the pair
  uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  uint8_t* staging = smem + kStages * Cfg::kStageBytes;
  uint64_t* bars = reinterpret_cast<uint64_t*>(staging + Cfg::kStagingBytes);
  uint64_t* full = bars;                                   // [kStages]  leader's: all bytes of the stage of both CTAs
  uint64_t* empty = bars + kStages;                        // [kStages]  local: consumed (commit to both CTAs)
  uint64_t* acc_full = bars + 2 * kStages;                 // [2]        local: accumulator complete (commit to both CTAs)
  uint64_t* acc_empty = bars + 2 * kStages + 2;            // [2]        leader's: drained by every epilogue warp of both CTAs
  uint64_t* drain = bars + 2 * kStages + 4;                // error path only
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 2 * kStages + 5);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const uint32_t cta = cluster_ctarank();                  // 0 = leader
  const int64_t pair = blockIdx.x >> 1;
  const int64_t num_pairs = gridDim.x >> 1;

  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) { mbar_init(&full[s], 1); mbar_init(&empty[s], 1); }
    for (int b = 0; b < 2; ++b) { mbar_init(&acc_full[b], 1); mbar_init(&acc_empty[b], 2 * Cfg::kEpilogueWarps); }
    mbar_init(drain, 1);
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(kTmemCols) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync_all();                                      // the peer's barriers exist before anything signals them
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  grid_dependency_wait();                                  // everything above touches shared and tensor memory only

  // (scalars of their own: a changed copy of the parameters was read back unchanged)
  int64_t M = p.M, K = p.K;
  if (p.live) {
    const int64_t n = load_count(p.live);
    if (p.live_is_k) K = n;
    else M = n;
  }
  const int64_t tiles_m = (M + 255) / 256;
  const int64_t tiles_n = (p.N + BN - 1) / BN;
  const int iters_all = (int)((K + 63) / 64);              // 0 where no row is left: the sums are zeros
  // a unit of work: a tile, or one split of the contraction of a tile (all tiles of a split, then the next: units that run together share operands)
  constexpr bool kSplit = kEpi == kEpiSumF32;
  const int64_t tiles = tiles_m * tiles_n, num_tiles = kSplit ? tiles * p.splits : tiles;

  if (warp == 0) {
    // ===== TMA producer (both CTAs): every copy reports to the leader's barrier =====
    int stage = 0;
    uint32_t phase = 0;
    bool ok = true;
    const uint32_t smem_base = smem_u32(smem);
    const uint32_t full_local = smem_u32(full);
    const uint32_t full_leader = map_to_cta(full_local, 0);
    for (int64_t tile = pair; tile < num_tiles && ok; tile += num_pairs) {
      int64_t tm, tn;
      const int split = kSplit ? (int)(tile / tiles) : 0, it0 = kSplit ? split * p.iters_per_split : 0;
      const int iters = kSplit && iters_all - it0 > p.iters_per_split ? p.iters_per_split : iters_all - it0;
      tile_coords(kSplit ? tile - split * tiles : tile, tiles_m, tiles_n, p.band, tm, tn);
      const int32_t m0 = (int32_t)(tm * 256 + cta * 128);             // this CTA's rows of A
      const int32_t n0 = (int32_t)(tn * BN + cta * 128);              // this CTA's rows of B
      for (int it = 0; it < iters; ++it) {
        ok = __all_sync(0xffffffffu, mbar_wait_cluster(&empty[stage], phase ^ 1u, abort_flag));
        if (!ok) {
          if (lane == 0) report(p.status, abort_flag, METIS_DEV_TIMEOUT_MMA);
          break;
        }
        const uint32_t sa = smem_base + stage * Cfg::kStageBytes;
        const uint32_t sb = sa + Cfg::kHalfBytes;
        const uint32_t bar = full_leader + stage * 8;
        const int32_t k0 = (it0 + it) * 64;
        if (elect_one()) {
          if (cta == 0) mbar_expect_tx_addr(full_local + stage * 8, 2 * Cfg::kStageBytes);
          if (kAMn) {
            tma_load_2d_pair(sa, &map_a, m0, k0, bar);
            tma_load_2d_pair(sa + Cfg::kBoxBytes, &map_a, m0 + 64, k0, bar);
          } else {
            tma_load_2d_pair(sa, &map_a, k0, m0, bar);
          }
          if (kBMn) {
            tma_load_2d_pair(sb, &map_b, n0, k0, bar);
            tma_load_2d_pair(sb + Cfg::kBoxBytes, &map_b, n0 + 64, k0, bar);
          } else {
            tma_load_2d_pair(sb, &map_b, k0, n0, bar);
          }
        }
        if (++stage == kStages) { stage = 0; phase ^= 1u; }
      }
    }
    grid_launch_dependents();                                // the last loads of this CTA are on their way: let the next kernel's CTAs in
  } else if (warp == 1) {
    // ===== tensor-core issuer (leader only) =====
    if (cta == 0 && iters_all > 0) {
      int stage = 0;
      uint32_t phase = 0, local_tile = 0;
      bool ok = true, issued = false;
      // descriptor low words: address, and for an MN-major tile the distance between its 64-element boxes as the leading byte offset;
      // one MMA takes 16 elements of the contraction: 32 bytes along a K-major row, 16 rows of an MN-major tile
      constexpr uint32_t a_lead = kAMn ? (uint32_t)(Cfg::kBoxBytes >> 4) : 1u, b_lead = kBMn ? (uint32_t)(Cfg::kBoxBytes >> 4) : 1u;
      constexpr uint32_t a_step = kAMn ? (16u * 128u) >> 4 : 2u, b_step = kBMn ? (16u * 128u) >> 4 : 2u;
      constexpr uint32_t idesc = idesc_bf16(BN, 256) | (kAMn ? (1u << 15) : 0u) | (kBMn ? (1u << 16) : 0u);
      const uint32_t smem_base = smem_u32(smem);
      const uint32_t empty_base = smem_u32(empty);
      for (int64_t tile = pair; tile < num_tiles && ok; tile += num_pairs, ++local_tile) {
        const uint32_t buf = local_tile & 1u;
        if (local_tile > 1) {
          ok = __all_sync(0xffffffffu, mbar_wait_cluster(&acc_empty[buf], ((local_tile >> 1) - 1u) & 1u, abort_flag));
          if (!ok) {
            if (lane == 0) report(p.status, abort_flag, METIS_DEV_TIMEOUT_EPI);
            break;
          }
        }
        tc_fence_after();
        const int it0 = kSplit ? (int)(tile / tiles) * p.iters_per_split : 0;
        const int iters = kSplit && iters_all - it0 > p.iters_per_split ? p.iters_per_split : iters_all - it0;
        const uint32_t d_tmem = tmem_base + buf * BN;
        for (int it = 0; it < iters; ++it) {
          ok = __all_sync(0xffffffffu, mbar_wait_cluster(&full[stage], phase, abort_flag));
          if (!ok) {
            if (lane == 0) report(p.status, abort_flag, METIS_DEV_TIMEOUT_TMA);
            break;
          }
          tc_fence_after();
          const uint32_t sa = smem_base + stage * Cfg::kStageBytes;
          const uint32_t a_lo = ((sa & 0x3FFFFu) >> 4) | (a_lead << 16);
          const uint32_t b_lo = (((sa + Cfg::kHalfBytes) & 0x3FFFFu) >> 4) | (b_lead << 16);
          if (elect_one()) {
#pragma unroll
            for (int j = 0; j < 4; ++j)
              tc_mma_bf16_pair(d_tmem, a_lo + a_step * j, b_lo + b_step * j, kOperandDescHi, idesc, (it > 0 || j > 0) ? 1u : 0u);
            tc_commit_pair(empty_base + stage * 8);
            if (it == iters - 1) tc_commit_pair(smem_u32(&acc_full[buf]));
          }
          issued = true;
          if (++stage == kStages) { stage = 0; phase ^= 1u; }
        }
      }
      if (!ok && issued && elect_one()) {
        // error path: let the tensor core finish what was issued before tensor memory is freed
        tc_commit_pair(smem_u32(drain));
        const uint64_t t0 = global_ns();
        while (!mbar_try(drain, 0) && global_ns() - t0 < kWaitLimitNs) {}
      }
      __syncwarp();
    }
  } else {
    // ===== epilogue (both CTAs): warps 2 to 9; warp w owns tensor-memory lanes 32*(w%4) .. +31 and 128 columns =====
    const int q = warp & 3;
    const int part = (warp - 2) >> 2;
    const uint32_t empty_leader = map_to_cta(smem_u32(acc_empty), 0);
    Staging st{staging + (warp - 2) * Cfg::kWarpBytes};
    // operands of the epilogue; `ahead` is the piece whose copies are on their way
    EpilogueOperand<kEpi == kEpiLinearOdd> gate = {p.gate, p.ldgate, p.gate_wide != 0, st.base + Cfg::kStores * 2048},
                                           residual = {p.residual, p.ldr, p.residual_wide != 0, gate.buf + Cfg::kPieceBytes};
    PieceAt ahead = {false, 0, 0};
    auto first_piece = [&](int64_t t) {                      // this warp's first piece of tile t
      int64_t tm = 0, tn = 0;
      if (t < num_tiles) tile_coords(t, tiles_m, tiles_n, p.band, tm, tn);
      PieceAt at = {t < num_tiles, tm * 256 + cta * 128 + q * 32, tn * BN + part * (32 * Cfg::kChunks)};
      at.valid = at.valid && at.row0 < M && at.col0 < p.N;
      return at;
    };
    const float alpha = kEpi == kEpiSum && p.gout ? common_weight(p.gout, p.inv_count, p.weight_scale) : 1.0f;
    uint32_t local_tile = 0;
    for (int64_t tile = pair; tile < num_tiles; tile += num_pairs, ++local_tile) {
      int64_t tm, tn;
      const int64_t split = kSplit ? tile / tiles : 0;
      tile_coords(kSplit ? tile - split * tiles : tile, tiles_m, tiles_n, p.band, tm, tn);
      const int64_t out0 = kSplit ? split * p.split_rows : 0;              // this split's first row of the sums
      const uint32_t buf = local_tile & 1u;
      const int64_t row0 = tm * 256 + cta * 128 + q * 32;
      const int64_t row = row0 + lane;
      const int64_t n0 = tn * BN + part * (32 * Cfg::kChunks);
      // warp-uniform: there are rows of this warp in the tile; the logits' gradient has zeros up to the next multiple of 64, what a stage of the
      // contraction over the rows reads
      const bool rows = row0 < (kEpi == kEpiGrad ? (M + 63) / 64 * 64 : M);
      int64_t hit = -1;                                    // the target's column in this launch
      float lse2 = 0.0f, weight = 0.0f, at_target = 0.0f;
      bool dead = true;
      if constexpr (kEpi == kEpiStats || kEpi == kEpiStatsEntropy || kEpi == kEpiGrad) {
        if (row < M) {
          const int64_t given = p.row_of ? p.row_of[row] : row;
          const int64_t t = p.target[given];
          if (t != p.ignore && t >= 0 && t < p.vocab) hit = t - p.col0;
          if constexpr (kEpi == kEpiGrad) {
            dead = t == p.ignore;
            lse2 = p.lse[given] * kLog2e;
            // (one gradient for all rows: it multiplies the products, not G, whose common factor bf16 would round)
            weight = p.gout_stride ? p.gout[given] * p.weight_scale : p.weight_scale < 0.0f ? -1.0f : 1.0f;
            if (t < 0 || t >= p.vocab) weight = NAN;       // (a target outside the vocabulary; ignored rows are dead)
            // The target's p - 1 from its log-probability, as the forward pass kept it: from this logit, which the tensor core cuts, and the one-hot
            // it would be off by 2e-6 of the logit, for a token that the model is sure of more than there is of it.
            if (hit >= n0 && hit < n0 + 32 * Cfg::kChunks) at_target = expm1f(p.target_logp[given]) * weight;
          }
        }
      }
      if constexpr (Cfg::kOperands) {
        if (rows && n0 < p.N && !ahead.valid) {
          gate.fetch(true, n0, row0, M, p.N);
          residual.fetch(true, n0, row0, M, p.N);
        }
        ahead.valid = false;
      }
      const bool sums = iters_all > 0;
      if (sums && !mbar_wait_cluster(&acc_full[buf], (local_tile >> 1) & 1u, abort_flag)) {
        if (lane == 0) report(p.status, abort_flag, METIS_DEV_TIMEOUT_MMA);
        break;
      }
      tc_fence_after();
      const uint32_t t_row = tmem_base + ((uint32_t)(q * 32) << 16) + buf * BN + part * (32 * Cfg::kChunks);
      RowStats stats = {-INFINITY, 0.0f, 0.0f};
      // the next chunk of the accumulator is read while this one is worked on, where the registers allow it
      constexpr bool kAhead = !Cfg::kOperands;
      uint32_t r[kAhead ? 2 : 1][32];
      if (kAhead && sums) tc_load32(t_row, r[0]);
      // (a piece with operands is some 600 instructions, several times that with the activations it may have: four copies of it leave the
      // instruction cache)
#pragma unroll(Cfg::kOperands ? 1 : Cfg::kChunks)
      for (int ch = 0; ch < Cfg::kChunks; ++ch) {
        uint32_t(&v)[32] = r[kAhead ? ch & 1 : 0];
        if (sums) {
          if (!kAhead) tc_load32(t_row + ch * 32, v);
          tc_wait_ld(v);
          if (ch < Cfg::kChunks - 1) {
            if (kAhead) tc_load32(t_row + (ch + 1) * 32, r[kAhead ? (ch + 1) & 1 : 0]);
          } else {
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive_cluster(empty_leader + buf * 8);
          }
        } else {
#pragma unroll
          for (int i = 0; i < 32; ++i) v[i] = 0u;
        }
        const int64_t col0 = n0 + ch * 32;
        if (rows && col0 < p.N) {
          const int64_t at = hit - col0;                   // the target's place in this chunk
          const bool here = at >= 0 && at < 32;
          if constexpr (kEpi == kEpiLinear) linear_chunk(p, st, &map_d, v, row0, col0);
          if constexpr (Cfg::kOperands) {
            PieceAt next = {ch + 1 < Cfg::kChunks && col0 + 32 < p.N, row0, col0 + 32};
            if (!next.valid) next = ahead = first_piece(tile + num_pairs);
            linear_wide_chunk(p, st, &map_d, &map_s, &map_act, gate, residual, v, row0, col0, next);
          }
          if constexpr (kEpi == kEpiStats || kEpi == kEpiStatsEntropy) {
            if (here) {                                    // (head_rows_kernel adds the target's)
#pragma unroll
              for (int i = 0; i < 32; ++i) if (at == i) v[i] = kMinusInfinity;
            }
            stats_chunk<kEpi == kEpiStatsEntropy>(p, stats, v, col0);
          }
          if constexpr (kEpi == kEpiGrad) {
            float g[32];
#pragma unroll
            for (int i = 0; i < 32; ++i) g[i] = exp2_fast(fmaf(__uint_as_float(v[i]), p.scale_log2e, -lse2)) * weight;
            if (here) {
#pragma unroll
              for (int i = 0; i < 32; ++i) if (at == i) g[i] = at_target;
            }
            uint32_t w[16];
#pragma unroll
            for (int i = 0; i < 16; ++i) w[i] = dead ? 0u : pack_bf16(g[2 * i], g[2 * i + 1]);
            if (p.half) {
              uint32_t low[16];                            // (what is left of an infinity is nothing)
#pragma unroll
              for (int i = 0; i < 16; ++i) {
                const float a = g[2 * i] - bf16_lo(w[i]), c = g[2 * i + 1] - bf16_hi(w[i]);
                low[i] = dead ? 0u : pack_bf16(fabsf(a) < INFINITY ? a : 0.0f, fabsf(c) < INFINITY ? c : 0.0f);
              }
              store_two_tma(st, &map_d, w, &map_s, low, (int32_t)col0, (int32_t)row0);
            } else {
              store_piece_tma(st, &map_d, w, (int32_t)col0, (int32_t)row0);
            }
          }
          if constexpr (kEpi == kEpiSum || kEpi == kEpiSumF32) {
            float g[32];
#pragma unroll
            for (int i = 0; i < 32; ++i) g[i] = kEpi == kEpiSum ? __uint_as_float(v[i]) * alpha : __uint_as_float(v[i]);
            if (kEpi == kEpiSumF32 && p.c && row < M) {
              const float* c = p.c + (out0 + row) * p.ldc + col0;
              if (col0 + 32 <= p.N) {
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                  const float4 f = *reinterpret_cast<const float4*>(c + 4 * i);
                  g[4 * i] += f.x; g[4 * i + 1] += f.y; g[4 * i + 2] += f.z; g[4 * i + 3] += f.w;
                }
              } else {
#pragma unroll
                for (int i = 0; i < 32; ++i) if (col0 + i < p.N) g[i] += c[i];
              }
            }
            uint32_t w[16];
            if constexpr (kEpi == kEpiSum) {
#pragma unroll
              for (int i = 0; i < 16; ++i) w[i] = pack_bf16(g[2 * i], g[2 * i + 1]);
              store_piece_tma(st, &map_d, w, (int32_t)col0, (int32_t)row0);
            } else {
#pragma unroll
              for (int h = 0; h < 2; ++h) {
#pragma unroll
                for (int i = 0; i < 16; ++i) w[i] = __float_as_uint(g[16 * h + i]);
                store_piece_tma(st, &map_d, w, (int32_t)col0 + 16 * h, (int32_t)(out0 + row0));
              }
            }
          }
        }
      }
      if constexpr (kEpi == kEpiStats || kEpi == kEpiStatsEntropy) {
        if (row < M) {
          const int64_t slot = (tn * 2 + part) * p.stats_ld + row;
          p.stats[slot] = make_float2(stats.m, stats.s);
          if constexpr (kEpi == kEpiStatsEntropy) p.stats_e[slot] = stats.e;
        }
      }
    }
    if constexpr (Cfg::kOperands) asm volatile("cp.async.wait_group 0;" ::: "memory");
    if (lane == 0) bulk_store_wait_all();                    // shared memory stays until the TMA unit has read it
  }

  tc_fence_before();
  __syncthreads();
  cluster_sync_all();                                      // nobody signals or reads the peer after this
  if (warp == 1) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(kTmemCols) : "memory");
  }
}

// ---- statistics of the pieces into losses ---------------------------------------------------------------------

// nll, lse and entropy of each row from the statistics of its `slots` pieces (slots of a row lie M apart).  The tensor core cuts what it adds
// up to instead of rounding it (16 products of a row at a time: 2e-6 of a logit at K = 3584), which shows in the target's logit, the largest
// of its row if the model knows anything.  So the pieces leave it out, and it is formed here, in fp32: log-probabilities of 16 rows of 3584 are
// 2.6e-7 from 64 bits instead of 2.2e-6.  With R, the others' sum, relative to the larger of the target's logit t and their maximum:
//   t the largest   -log p = log(1 + R), log1p: for a token the model is sure of (1 - p of 1e-6) as many bits of it as of any, and never negative
//   otherwise       -log p = log(R + 2^d) - d ln 2, d = t less their maximum; R is 1 at least and d negative
//   kRows = 32  a block of 32 warps takes 32 rows: its warps take the slots in turn, neighbouring lanes neighbouring rows
//   kRows = 1   few rows: a block of 8 warps takes one, its threads the slots
struct HeadRows {
  const float2* stats;  const float* stats_e;
  const __nv_bfloat16* h;  int64_t ldh;                    // rows as the statistics have them (packed or not)
  const __nv_bfloat16* w;  int64_t ldw;
  const int64_t* target;  int64_t ignore, vocab, M;
  const int32_t* row_of;  const int32_t* live;
  int32_t pieces, slots;                                   // 16-byte pieces of a row of h; slots
  float scale, scale_log2e, sign;
  float* nll;  float* lse;  float* entropy;  float* target_logp;      // the last two may be null
};

__device__ __forceinline__ float dot8(uint4 a, uint4 b, float c) {
  const uint32_t x[4] = {a.x, a.y, a.z, a.w}, y[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) c = fmaf(bf16_hi(x[i]), bf16_hi(y[i]), fmaf(bf16_lo(x[i]), bf16_lo(y[i]), c));
  return c;
}
__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

template <bool kEntropy, int kRows>
__global__ void __launch_bounds__(kRows == 32 ? 1024 : 256)
head_rows_kernel(const HeadRows p) {
  grid_dependency_wait();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  constexpr int kWarps = kRows == 32 ? 32 : 8;
  __shared__ RowStats s_part[kWarps][32];
  __shared__ float s_dot[32];
  const int64_t rows = p.live ? load_count(p.live) : p.M, row0 = (int64_t)blockIdx.x * kRows;
  if (row0 >= rows) return;
  // the row's target, or -1 where none is to be looked up
  auto target_of = [&](int64_t row) {
    const int64_t t = p.target[p.row_of ? p.row_of[row] : row];
    return t != p.ignore && t >= 0 && t < p.vocab ? t : (int64_t)-1;
  };
  // a warp has a row, or a part of the block's
  {
    const int64_t row = kRows == 32 ? row0 + warp : row0, t = row < rows ? target_of(row) : -1;
    float dot = 0.0f;
    if (t >= 0) {
      const uint4 *hp = reinterpret_cast<const uint4*>(p.h + row * p.ldh), *wp = reinterpret_cast<const uint4*>(p.w + t * p.ldw);
#pragma unroll 4
      for (int k = kRows == 32 ? lane : (int)threadIdx.x; k < p.pieces; k += kRows == 32 ? 32 : 256) dot = dot8(hp[k], wp[k], dot);
    }
    dot = warp_sum(dot);
    if (lane == 0) s_dot[warp] = dot;
  }

  RowStats a = {-INFINITY, 0.0f, 0.0f};
  const int64_t row = kRows == 32 ? row0 + lane : row0;
  if (row < rows) {
    constexpr int kFly = 8, kStep = kRows == 32 ? kWarps : 256;         // loads in flight
    for (int s0 = kRows == 32 ? warp : (int)threadIdx.x; s0 < p.slots; s0 += kStep * kFly) {
      float2 v[kFly];
      float e[kFly];
#pragma unroll
      for (int i = 0; i < kFly; ++i) {
        const int s = s0 + kStep * i;
        v[i] = make_float2(-INFINITY, 0.0f);
        e[i] = 0.0f;
        if (s < p.slots) {
          v[i] = p.stats[(int64_t)s * p.M + row];
          if constexpr (kEntropy) e[i] = p.stats_e[(int64_t)s * p.M + row];
        }
      }
#pragma unroll
      for (int i = 0; i < kFly; ++i) stats_merge<kEntropy>(a, RowStats{v[i].x, v[i].y, e[i]});
    }
  }
  if constexpr (kRows == 1) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      RowStats b;
      b.m = __shfl_xor_sync(0xffffffffu, a.m, o);
      b.s = __shfl_xor_sync(0xffffffffu, a.s, o);
      b.e = kEntropy ? __shfl_xor_sync(0xffffffffu, a.e, o) : 0.0f;
      if (lane & o) { const RowStats t = a; a = b; b = t; }            // the same order on both sides
      stats_merge<kEntropy>(a, b);
    }
  }
  s_part[warp][lane] = a;
  __syncthreads();
  if (warp == 0 && row < rows && (kRows == 32 || lane == 0)) {
    for (int w = 1; w < kWarps; ++w) stats_merge<kEntropy>(a, s_part[w][lane]);
    const int64_t given = p.row_of ? p.row_of[row] : row, t = p.target[given];
    const bool ignored = t == p.ignore, inside = t >= 0 && t < p.vocab;
    float nll = NAN, log_sum;
    if (!ignored && inside) {
      float l2 = 0.0f;                                     // the target's logit, times log2 e
      if constexpr (kRows == 32) {
        l2 = s_dot[lane];
      } else {
#pragma unroll
        for (int w = 0; w < 8; ++w) l2 += s_dot[w];
      }
      l2 *= p.scale_log2e;
      const float base = stats_base(fmaxf(a.m, l2)), rest = a.s * exp2_fast(a.m - base), d = l2 - base;
      log_sum = d == 0.0f ? log1pf(rest) : logf(rest + exp2_fast(d));
      nll = log_sum - kLn2 * d;
      stats_merge<kEntropy>(a, RowStats{l2, 1.0f, 0.0f});
    } else {
      log_sum = logf(a.s);
    }
    p.lse[given] = fmaf(a.m, kLn2, log_sum);
    p.nll[given] = ignored ? 0.0f : p.sign * nll;
    if (p.target_logp) p.target_logp[given] = -nll;
    // H = log s - sum p (l - m): p = 2^(l - m) / s, l - m in units of log2
    if constexpr (kEntropy) p.entropy[given] = ignored ? 0.0f : log_sum - kLn2 * (a.e / a.s);
  }
}

// The same from lse alone, for a backward pass that was not given what the forward pass had: to 2^-24 of the logit.  A warp has a row.
__global__ void __launch_bounds__(256)
head_target_kernel(const __nv_bfloat16* h, int64_t ldh, const __nv_bfloat16* w, int64_t ldw, const int64_t* target, int64_t ignore, int64_t vocab, int64_t M,
                   int pieces, float scale, const float* lse, float* target_logp) {
  grid_dependency_wait();
  const int lane = threadIdx.x & 31;
  for (int64_t row = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5); row < M; row += (int64_t)gridDim.x * 8) {
    const int64_t t = target[row];
    if (t == ignore || t < 0 || t >= vocab) continue;
    const uint4 *hp = reinterpret_cast<const uint4*>(h + row * ldh), *wp = reinterpret_cast<const uint4*>(w + t * ldw);
    float dot = 0.0f;
#pragma unroll 4
    for (int k = lane; k < pieces; k += 32) dot = dot8(hp[k], wp[k], dot);
    dot = warp_sum(dot);
    if (lane == 0) target_logp[row] = fmaf(dot, scale, -lse[row]);
  }
}

// ---- rows that are not ignored -----------------------------------------------------------------------------------
// A third of the tokens of a training batch and more are prompt or padding.  Where the products behind are long enough (kPackFlops), the
// others are brought together first: 8192 rows, a third ignored, 151936 x 1536 with gradients 11.6 ms, 8.0 so.

// row_of[i] = the i-th row that is not ignored, place_of[m] = its i or -1, *live = their number; zeros for the losses of the others.  One block,
// in the order of the rows.
__global__ void __launch_bounds__(1024)
head_index_kernel(const int64_t* target, int64_t ignore, int64_t M, int32_t* row_of, int32_t* place_of,
                  int32_t* live, float* nll, float* entropy) {
  grid_dependency_wait();
  __shared__ int s_warp[2][32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int before = 0;
  for (int64_t m0 = 0, it = 0; m0 < M; m0 += 1024, ++it) {
    const int64_t m = m0 + threadIdx.x;
    const bool on = m < M && target[m] != ignore;
    const uint32_t mask = __ballot_sync(0xffffffffu, on);
    int* counts = s_warp[it & 1];
    if (lane == 0) counts[warp] = __popc(mask);
    __syncthreads();
    int total = counts[lane], mine = lane < warp ? total : 0;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      total += __shfl_xor_sync(0xffffffffu, total, o);
      mine += __shfl_xor_sync(0xffffffffu, mine, o);
    }
    const int place = before + mine + __popc(mask & ((1u << lane) - 1u));
    if (m < M) {
      place_of[m] = on ? place : -1;
      if (on) {
        row_of[place] = (int32_t)m;
      } else {
        if (nll) nll[m] = 0.0f;
        if (entropy) entropy[m] = 0.0f;
      }
    }
    before += total;
  }
  if (threadIdx.x == 0) *live = before;
}

// packed[i] = h[row_of[i]], and zeros up to the next multiple of 64 (what a stage of the contraction over the rows reads); rows of 16-byte pieces
__global__ void __launch_bounds__(256)
head_gather_kernel(const __nv_bfloat16* h, int64_t ldh, int64_t M, int pieces, const int32_t* row_of, const int32_t* live,
                   __nv_bfloat16* packed) {
  grid_dependency_wait();
  const int64_t n = load_count(live), end = (n + 63) / 64 * 64 < M ? (n + 63) / 64 * 64 : M;
  for (int64_t i = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5); i < end; i += (int64_t)gridDim.x * 8) {
    uint4* to = reinterpret_cast<uint4*>(packed) + i * pieces;
    if (i < n) {
      const uint4* from = reinterpret_cast<const uint4*>(h + row_of[i] * ldh);
#pragma unroll 4
      for (int k = threadIdx.x & 31; k < pieces; k += 32) to[k] = from[k];
    } else {
      for (int k = threadIdx.x & 31; k < pieces; k += 32) to[k] = make_uint4(0u, 0u, 0u, 0u);
    }
  }
}

// The rows of x `parts` times, `half` apart and zeros between: what a gradient of two parts is contracted with.  With `target`, zeros in the rows
// that are ignored: their gradient is 0, but 0 times what they may hold (a NaN of the padding) is not.
__global__ void __launch_bounds__(256)
stack_rows_kernel(const __nv_bfloat16* x, int64_t ldx, int64_t M, int parts, int64_t half, int64_t pieces, const int64_t* target, int64_t ignore, __nv_bfloat16* out) {
  grid_dependency_wait();
  for (int64_t e = (int64_t)blockIdx.x * 256 + threadIdx.x; e < parts * half * pieces; e += (int64_t)gridDim.x * 256) {
    const int64_t i = e / pieces, k = e - i * pieces, m = i < half ? i : i - half;
    reinterpret_cast<uint4*>(out)[e] = m < M && !(target && target[m] == ignore) ? reinterpret_cast<const uint4*>(x + m * ldx)[k] : make_uint4(0u, 0u, 0u, 0u);
  }
}

// d[m] = alpha times the sum over the splits of row place_of[m] of the sums (m itself where there is no place_of) and of the row `half` behind
// it (0: none), in bf16; zeros for a place of -1.  A thread takes eight columns of a row.
__global__ void __launch_bounds__(256)
finish_sums_kernel(const float* sums, int splits, int64_t split_rows, int64_t M, int pieces, const int32_t* place_of, int64_t half, const float* gout, const float* inv_count,
                   float scale, __nv_bfloat16* d, int64_t ldd) {
  grid_dependency_wait();
  const float alpha = gout ? common_weight(gout, inv_count, scale) : 1.0f;
  const int64_t ld = 8 * (int64_t)pieces, total = M * pieces;
  for (int64_t e = (int64_t)blockIdx.x * 256 + threadIdx.x; e < total; e += (int64_t)gridDim.x * 256) {
    const int64_t m = e / pieces, k = e - m * pieces, i = place_of ? place_of[m] : m;
    float v[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
    if (i >= 0) {
#pragma unroll 4
      for (int s = 0; s < splits; ++s) {
        const float4* at = reinterpret_cast<const float4*>(sums + (s * split_rows + i) * ld + 8 * k);
        const float4 x = at[0], y = at[1];
        v[0] += x.x; v[1] += x.y; v[2] += x.z; v[3] += x.w;
        v[4] += y.x; v[5] += y.y; v[6] += y.z; v[7] += y.w;
        if (half) {
          const float4 z = at[half * (ld / 4)], u = at[half * (ld / 4) + 1];
          v[0] += z.x; v[1] += z.y; v[2] += z.z; v[3] += z.w;
          v[4] += u.x; v[5] += u.y; v[6] += u.z; v[7] += u.w;
        }
      }
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] *= alpha;
    reinterpret_cast<uint4*>(d + m * ldd)[k] = pack8(v);
  }
}

// loss = sum of nll, or that over the number of rows that are not ignored; inv_count = 1 / that number (1 for the sum).  One block,
// fixed order.
__global__ void __launch_bounds__(1024)
head_sum_kernel(const float* nll, const int64_t* target, int64_t ignore, int64_t M, int mean,
                float* loss, float* inv_count) {
  grid_dependency_wait();
  __shared__ double s_sum[32];
  __shared__ unsigned long long s_count[32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  double sum = 0.0;
  unsigned long long count = 0;
  for (int64_t i = threadIdx.x; i < M; i += 1024) {
    sum += (double)nll[i];
    count += target[i] != ignore;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    sum += __shfl_xor_sync(0xffffffffu, sum, o);
    count += __shfl_xor_sync(0xffffffffu, count, o);
  }
  if (lane == 0) { s_sum[warp] = sum; s_count[warp] = count; }
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < 32; ++w) { sum += s_sum[w]; count += s_count[w]; }
    *loss = (float)(mean ? sum / (double)count : sum);     // (no row at all: 0 / 0, as torch has it)
    *inv_count = !mean ? 1.0f : count ? (float)(1.0 / (double)count) : 0.0f;       // (then there is no gradient either)
  }
}

// ---- backward of the epilogue -----------------------------------------------------------------------------------

// Eight consecutive elements at any address (of which `left` are in the row): the one or two aligned 16 bytes that hold them, shifted.  What
// lies beside the row in them belongs to the same allocation and is not used.
template <bool kWide> __device__ __forceinline__ void load8_any(const __nv_bfloat16* at, int64_t left, float (&v)[8]) {
  if constexpr (kWide) {
    const uint4 w = *reinterpret_cast<const uint4*>(at);
    v[0] = bf16_lo(w.x); v[1] = bf16_hi(w.x); v[2] = bf16_lo(w.y); v[3] = bf16_hi(w.y);
    v[4] = bf16_lo(w.z); v[5] = bf16_hi(w.z); v[6] = bf16_lo(w.w); v[7] = bf16_hi(w.w);
  } else {
    const uintptr_t a = reinterpret_cast<uintptr_t>(at);
    const uint32_t off = (uint32_t)(a & 15);
    const int64_t bytes = 2 * (left < 8 ? left : 8);
    const uint4* p = reinterpret_cast<const uint4*>(a & ~(uintptr_t)15);
    const uint4 lo = p[0];
    uint4 hi = make_uint4(0u, 0u, 0u, 0u);
    if (off + bytes > 16) hi = p[1];
    uint32_t x[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
#pragma unroll
    for (int k = 0; k < 6; ++k) x[k] = (off & 8) ? x[k + 2] : x[k];
#pragma unroll
    for (int k = 0; k < 5; ++k) x[k] = (off & 4) ? x[k + 1] : x[k];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const uint32_t w = __funnelshift_r(x[k], x[k + 1], (off & 2) * 8);
      v[2 * k] = bf16_lo(w);
      v[2 * k + 1] = bf16_hi(w);
    }
  }
}
// The eight elements of every lane, 256 together, to a run of `count` elements at any address: through the warp's buffer, laid out there as the
// run lies to 16 bytes, so that all but its two ends leave as whole 16 bytes.
__device__ __forceinline__ void store_run(__nv_bfloat16* run, int count, unsigned short* buf, const float (&v)[8]) {
  const int lane = threadIdx.x & 31, off = (int)(reinterpret_cast<uintptr_t>(run) & 15) >> 1;
  const uint4 q = pack8(v);
  const uint32_t w[4] = {q.x, q.y, q.z, q.w};
  __syncwarp();
#pragma unroll
  for (int i = 0; i < 8; ++i) buf[off + lane * 8 + i] = (unsigned short)(w[i >> 1] >> ((i & 1) * 16));
  __syncwarp();
  unsigned short* to = reinterpret_cast<unsigned short*>(run) - off;
  for (int k = lane; k * 8 < off + count; k += 32) {
    if (k * 8 >= off && k * 8 + 8 <= off + count) {
      *reinterpret_cast<uint4*>(to + k * 8) = *reinterpret_cast<const uint4*>(buf + k * 8);
    } else {
      for (int i = k * 8; i < k * 8 + 8; ++i) if (i >= off && i < off + count) to[i] = buf[i];
    }
  }
}

// dz = dy * gate * slope, dgate = dy * act, and column sums of dz before its rounding.  A warp's lane has eight columns of a row, the
// block's eight warps take eight rows at a time; a block owns 256 columns and every gridDim.y-th group of rows.  dz, slope and act have
// 16-byte aligned rows; kWide: all the others do too, and N is a multiple of 8.  Bound by memory: 8192 x 8960 with gate 145 us, 6.1 TB/s.
template <bool kWide>
__global__ void __launch_bounds__(256)
linear_pointwise_kernel(const __nv_bfloat16* dy, int64_t lddy, const __half* slope, int64_t lds, const __nv_bfloat16* act, int64_t lda,
                        const __nv_bfloat16* gate, int64_t ldgate, int64_t M, int64_t N,
                        __nv_bfloat16* dz, int64_t lddz, int64_t half, __nv_bfloat16* dgate, int64_t lddg,
                        float* sums) {
  grid_dependency_wait();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t col0 = (int64_t)blockIdx.x * 256, col = col0 + lane * 8, left = N - col;
  const int count = N - col0 < 256 ? (int)(N - col0) : 256;
  __shared__ __align__(16) unsigned short s_run[8][264];
  float acc[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) acc[i] = 0.0f;
  for (int64_t row = (int64_t)blockIdx.y * 8 + warp; row < (half ? half : M); row += (int64_t)gridDim.y * 8) {
    float d[8], a[8], out[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) { d[i] = 0.0f; a[i] = 0.0f; out[i] = 0.0f; }
    if (left > 0 && row < M) {
      float g[8];
      uint4 s;
      load8_any<kWide>(dy + row * lddy + col, left, d);
      if (slope) s = *reinterpret_cast<const uint4*>(slope + row * lds + col);
      if (dgate) load8_any<true>(act + row * lda + col, left, a);
      if (gate) load8_any<kWide>(gate + row * ldgate + col, left, g);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        out[i] = d[i];
        if (slope) out[i] *= (1.0f / kSlopeScale) * __half2float(reinterpret_cast<const __half*>(&s)[i]);
        if (gate) out[i] *= g[i];
        a[i] *= d[i];
        acc[i] += out[i];
      }
    }
    if (left > 0) {
      for (int part = 0; dz && part < (half ? 2 : 1); ++part) {
        __nv_bfloat16* to = dz + (part * half + row) * lddz + col;
        const uint4 q = pack8(out);
        if (kWide || left >= 8) *reinterpret_cast<uint4*>(to) = q;
        else for (int i = 0; i < left; ++i) to[i] = __float2bfloat16_rn(out[i]);
        const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
        for (int i = 0; i < 8; ++i) {                      // what the first part leaves (of an infinity nothing)
          const float r = out[i] - (i & 1 ? bf16_hi(w[i >> 1]) : bf16_lo(w[i >> 1]));
          out[i] = fabsf(r) < INFINITY ? r : 0.0f;
        }
      }
      if (kWide && dgate && row < M) *reinterpret_cast<uint4*>(dgate + row * lddg + col) = pack8(a);
    }
    if (!kWide && dgate && row < M) store_run(dgate + row * lddg + col0, count, s_run[warp], a);
  }
  if (sums) {
    __shared__ float s_sum[8][256];
#pragma unroll
    for (int i = 0; i < 8; ++i) s_sum[warp][lane * 8 + i] = acc[i];
    __syncthreads();
    const int c = threadIdx.x;
    float t = s_sum[0][c];
#pragma unroll
    for (int w = 1; w < 8; ++w) t += s_sum[w][c];
    if (col0 + c < N) sums[(int64_t)blockIdx.y * N + col0 + c] = t;
  }
}

template <typename T>
__global__ void __launch_bounds__(256)
linear_bias_kernel(const float* sums, int groups, int64_t N, T* out) {
  grid_dependency_wait();
  const int64_t c = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (c >= N) return;
  float t = 0.0f;
#pragma unroll 8
  for (int g = 0; g < groups; ++g) t += sums[(int64_t)g * N + c];
  if constexpr (sizeof(T) == 2) out[c] = __float2bfloat16_rn(t);
  else out[c] = t;
}

// ---- host side ------------------------------------------------------------------------------------------------

static int32_t check_rows(const void* p, int64_t ld, int64_t cols, const char* what) {
  if (!p) return fail(METIS_ERR_BAD_ARGUMENT, "%s is null", what);
  if (!aligned16(p) || ld < cols || ld % 8 != 0) return fail(METIS_ERR_BAD_ALIGNMENT, "%s must be 16-byte aligned with a leading dimension that is a multiple of 8", what);
  return METIS_OK;
}
// coordinates of a copy are 32 bits
static int32_t check_extent(int64_t n, const char* what) {
  if (n <= 0) return fail(METIS_ERR_BAD_SHAPE, "%s = %lld must be positive", what, (long long)n);
  if (n >= ((int64_t)1 << 31) - 512) return fail(METIS_ERR_TOO_LARGE, "%s = %lld does not fit 32 bits", what, (long long)n);
  return METIS_OK;
}

// blocks of eight warps for so many warps' work
static unsigned row_blocks(int64_t warps) {
  const int64_t blocks = ceil_div(warps, 8), most = (int64_t)device_sm_count() * 8;
  return (unsigned)(blocks < most ? blocks : most);
}

struct DenseOperand {
  const void* p;
  int64_t ld;
  bool mn;                                                 // the contraction lies in the rows
};

template <bool kAMn, bool kBMn, int kEpi>
static int32_t launch_dense(const DenseOperand& a, const DenseOperand& b, const CUtensorMap& map_d, DenseParams p, cudaStream_t st, const CUtensorMap& map_s = {}, const CUtensorMap& map_act = {}) {
  using Cfg = DenseCfg<kEpi>;
  const CUtensorMapDataType dt = CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  CUtensorMap ma, mb;
  if (kAMn) { if (int32_t rc = make_map(&ma, dt, 2, a.p, p.M, p.K, a.ld * 2, 64, 64, "A (MN-major)")) return rc; }
  else      { if (int32_t rc = make_map(&ma, dt, 2, a.p, p.K, p.M, a.ld * 2, 64, 128, "A (K-major)")) return rc; }
  if (kBMn) { if (int32_t rc = make_map(&mb, dt, 2, b.p, p.N, p.K, b.ld * 2, 64, 64, "B (MN-major)")) return rc; }
  else      { if (int32_t rc = make_map(&mb, dt, 2, b.p, p.K, p.N, b.ld * 2, 64, 128, "B (K-major)")) return rc; }
  p.band = 16;                                             // (4, 8, 16, 32: loss of 2048 tokens over 151936 x 1536 774, 770, 755, 746 us; linear layers the same)
  if (p.splits < 1) p.splits = 1;
  if (p.splits == 1) p.iters_per_split = INT32_MAX;
  const int64_t tiles = ceil_div(p.M, 256) * ceil_div(p.N, 256) * p.splits;
  int64_t pairs = device_sm_count() / 2;
  if (pairs > tiles) pairs = tiles;
  if (!p.live) pairs = ceil_div(tiles, ceil_div(tiles, pairs));        // the fewest that finish in the same number of rounds
  auto kern = dense_gemm_pair_kernel<kAMn, kBMn, kEpi>;
  static std::atomic<uint64_t> done{0};
  METIS_CUDA_OK(allow_shared(reinterpret_cast<const void*>(kern), Cfg::kSmemBytes, done));
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(2 * pairs), 1, 1);
  cfg.blockDim = dim3(Cfg::kThreads, 1, 1);
  cfg.dynamicSmemBytes = Cfg::kSmemBytes;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 2;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = launch_overlap_enabled(kLaunchGemm) ? 2 : 1;
  METIS_CUDA_OK(cudaLaunchKernelEx(&cfg, kern, ma, mb, map_d, map_s, map_act, p));
  dense_launches.fetch_add(1, std::memory_order_relaxed);
  return METIS_OK;
}

// pieces of 32 rows x 64 bytes that the epilogue stores
static int32_t map_bf16(CUtensorMap* map, const void* d, int64_t ld, int64_t M, int64_t N, const char* what) {
  return make_map(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, d, N, M, ld * 2, 32, 32, what, 64);
}

// D = A B^T for gradients: (A K-major, B MN-major), or (both MN-major).  In bf16; or `sums`, fp32 [splits, split_rows, N] with split_rows = M in
// whole tiles, added to what they hold where `add` is set, and finish_sums behind them.
struct CommonWeight {                                      // what a bf16 D is multiplied by: scale * *gout * (inv_count ? *inv_count : 1); nothing where gout is null
  const float* gout = nullptr;
  const float* inv_count = nullptr;
  float scale = 1.0f;
};
struct Splits {
  int32_t splits, iters_per_split;
  int64_t rows, bytes;                                     // of the sums
};
static int32_t dense_sum(const DenseOperand& a, const DenseOperand& b, int64_t M, int64_t N, int64_t K, void* d, int64_t ldd, int32_t* status, cudaStream_t st,
                         const int32_t* live = nullptr, const Splits* sp = nullptr, float* sums = nullptr, bool add = false, const CommonWeight& weight = {}) {
  DenseParams p = {};
  p.gout = weight.gout; p.inv_count = weight.inv_count; p.weight_scale = weight.scale;
  p.live = live; p.live_is_k = a.mn;                       // (rows that are not ignored: the output's, or those a weight's gradient sums over)
  p.M = M; p.N = N; p.K = K; p.status = status;
  CUtensorMap md = {};
  if (sums) {
    p.splits = sp->splits; p.iters_per_split = sp->iters_per_split; p.split_rows = sp->rows;
    p.c = add ? sums : nullptr; p.ldc = N;
    if (int32_t rc = make_map(&md, CU_TENSOR_MAP_DATA_TYPE_FLOAT32, 4, sums, N, sp->splits * sp->rows, N * 4, 16, 32, "sums", 64)) return rc;
    return a.mn ? launch_dense<true, true, kEpiSumF32>(a, b, md, p, st) : launch_dense<false, true, kEpiSumF32>(a, b, md, p, st);
  }
  if (int32_t rc = map_bf16(&md, d, ldd, M, N, "D")) return rc;
  return a.mn ? launch_dense<true, true, kEpiSum>(a, b, md, p, st) : launch_dense<false, true, kEpiSum>(a, b, md, p, st);
}

// Splits of the contraction: what fills the rounds of pairs, weighed against the sums' way through memory (0.29 us for a stage of a round, 5
// TB/s; fewer than 8 stages to a split are not worth its start).  Loss's input gradient, us, one / so many: 1021 x 1000 over 32003 224 / 69 (4),
// 2048 x 1536 over 75968 374 / 268 (3).
static Splits plan_splits(int64_t M, int64_t N, int64_t K) {
  const int64_t tiles = ceil_div(M, 256) * ceil_div(N, 256), iters = ceil_div(K, 64), pairs = device_sm_count() / 2;
  Splits best = {1, (int32_t)iters, ceil_div(M, 256) * 256, 0};
  float best_us = 0.29f * (float)(ceil_div(tiles, pairs) * iters) * 0.95f;
  for (int s = 2; s <= 16; ++s) {
    const int64_t per = ceil_div(iters, s);
    if (per < 8 || ceil_div(iters, per) != s) continue;
    const float us = 0.29f * (float)(ceil_div(tiles * s, pairs) * per) + 5.0f + (float)(8 * s * best.rows * N) / 5e6f;
    if (us < best_us) {
      best_us = us;
      best.splits = s;
      best.iters_per_split = (int32_t)per;
    }
  }
  best.bytes = best.splits * best.rows * N * 4;
  return best;
}

// Whether a product goes to the kernel for few tokens, with the shape it takes there: by a model of both.  A round of 256 x 256 tiles takes
// 0.29 us for each stage of the contraction, and its start, end and launch 7.5 us; a quarter of the pairs or less of them busy is what it
// loses by (3584 x 18944: 92 us for 1 to 256 tokens).
static bool few_tokens(int64_t M, int64_t N, int64_t K, bool w_mn, SmallShape* sh) {
  if (M > 2048) return false;
  const SmallPlan plan = plan_dense_small(M, N, K, w_mn);
  *sh = plan.sh;
  const int64_t pairs = device_sm_count() / 2, tiles = ceil_div(M, 256) * ceil_div(N, 256), rounds = ceil_div(tiles, pairs);
  const float busy = tiles < pairs ? (float)tiles / (float)pairs : 1.0f;             // (the weight comes to the pairs that have a tile)
  const float tiles_us = 0.29f * (float)(rounds * ceil_div(K, 64)), memory_us = (float)(2 * N * K) / (5.5e6f * busy);
  const float pair_us = 7.5f + (tiles_us > memory_us ? tiles_us : memory_us);
#ifdef METIS_TIMING_KNOBS
  if (const char* e = getenv("METIS_DEV_DENSE_SMALL")) return atoi(e) != 0;
  if (getenv("METIS_DEV_DENSE_PRINT")) fprintf(stderr, "M %lld N %lld K %lld: small %.1f (rows %d bn %d kb %d splits %d stages %d) pair %.1f\n", (long long)M, (long long)N, (long long)K, plan.us, plan.sh.rows, plan.sh.bn, plan.sh.kb, plan.sh.splits, plan.sh.stages, pair_us);
#endif
  return plan.us < pair_us;
}

// Columns of the vocabulary that the backward pass takes at a time: their gradients G [M, columns] in bf16 go through memory.  Loss and
// gradients of 8192 x 151936 x 1536 with pieces of 256 MiB 12.9 ms, of 512 12.3, of 1024 12.3, whole 12.2.
constexpr int64_t kPieceBytes = (int64_t)512 << 20;
static int64_t piece_columns(int64_t M, int64_t V) {
  int64_t columns = kPieceBytes / (2 * M) / 256 * 256;
  if (columns < 256) columns = 256;
  if (columns >= V) return ceil_div(V, 8) * 8;
  return ceil_div(ceil_div(V, ceil_div(V, columns)), 256) * 256;       // pieces of one size
}

}  // namespace metis

using namespace metis;

extern "C" int64_t metis_dense_launches(void) { return dense_launches.load(std::memory_order_relaxed); }

extern "C" int32_t metis_linear(const metis_linear_args* a) {
  if (!a) return fail(METIS_ERR_BAD_ARGUMENT, "args is null");
  if (int32_t rc = check_extent(a->M, "M")) return rc;
  if (int32_t rc = check_extent(a->N, "N")) return rc;
  if (int32_t rc = check_extent(a->K, "K")) return rc;
  if (a->K % 8 != 0) return fail(METIS_ERR_BAD_SHAPE, "K = %lld must be a multiple of 8", (long long)a->K);
  if (a->activation < METIS_ACT_NONE || a->activation > METIS_ACT_GELU_TANH) return fail(METIS_ERR_BAD_ARGUMENT, "unknown activation %d", a->activation);
  if (a->bias && a->bias_dtype != METIS_DTYPE_BF16 && a->bias_dtype != METIS_DTYPE_F32) return fail(METIS_ERR_BAD_ARGUMENT, "unknown bias_dtype %d", a->bias_dtype);
  if (int32_t rc = check_rows(a->x, a->ldx, a->K, "x")) return rc;
  if (int32_t rc = check_rows(a->w, a->ldw, a->K, "w")) return rc;
  if (!a->y) return fail(METIS_ERR_BAD_ARGUMENT, "y is null");
  if (a->slope && a->activation == METIS_ACT_NONE) return fail(METIS_ERR_BAD_ARGUMENT, "slope is given without an activation");
  if (a->act) if (int32_t rc = check_rows(a->act, a->ldact, a->N, "act")) return rc;
  if (a->slope) if (int32_t rc = check_rows(a->slope, a->ldslope, a->N, "slope")) return rc;
  const uintptr_t odd = reinterpret_cast<uintptr_t>(a->y) | reinterpret_cast<uintptr_t>(a->gate) | reinterpret_cast<uintptr_t>(a->residual);
  if ((odd & 1u) || (reinterpret_cast<uintptr_t>(a->bias) & (a->bias_dtype == METIS_DTYPE_F32 ? 3u : 1u)))
    return fail(METIS_ERR_BAD_ALIGNMENT, "a tensor is not aligned to its elements");
  if (a->ldy < a->N || (a->gate && a->ldgate < a->N) || (a->residual && a->ldr < a->N))
    return fail(METIS_ERR_BAD_ARGUMENT, "a leading dimension is smaller than N = %lld", (long long)a->N);
  DenseParams p = {};
  p.M = a->M; p.N = a->N; p.K = a->K; p.status = a->status;
  p.bias = a->bias; p.bias_f32 = a->bias_dtype == METIS_DTYPE_F32; p.act = a->activation;
  auto wide = [](const void* t, int64_t ld) { return t && aligned16(t) && ld % 8 == 0; };
  p.gate = static_cast<const __nv_bfloat16*>(a->gate); p.ldgate = a->ldgate; p.gate_wide = wide(a->gate, a->ldgate);
  p.residual = static_cast<const __nv_bfloat16*>(a->residual); p.ldr = a->ldr; p.residual_wide = wide(a->residual, a->ldr);
  p.d = static_cast<__nv_bfloat16*>(a->y); p.ldd = a->ldy; p.d_wide = wide(a->y, a->ldy);
  p.act_out = static_cast<__nv_bfloat16*>(a->act); p.ldact = a->ldact;
  p.slope = static_cast<uint32_t*>(a->slope); p.ldslope = a->ldslope;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(a->stream);
  SmallShape sh;
  if (few_tokens(a->M, a->N, a->K, false, &sh)) return launch_dense_small(sh, a->x, a->ldx, a->w, false, a->ldw, p, st);
  const DenseOperand x = {a->x, a->ldx, false}, w = {a->w, a->ldw, false};
  CUtensorMap md = {}, ms = {}, ma = {};
  if (p.d_wide) if (int32_t rc = map_bf16(&md, a->y, a->ldy, a->M, a->N, "y")) return rc;
  if (a->slope) if (int32_t rc = map_bf16(&ms, a->slope, a->ldslope, a->M, a->N, "slope")) return rc;        // (16 bits are 16 bits)
  if (a->act) if (int32_t rc = map_bf16(&ma, a->act, a->ldact, a->M, a->N, "act")) return rc;
  if ((a->gate && !p.gate_wide) || (a->residual && !p.residual_wide)) return launch_dense<false, false, kEpiLinearOdd>(x, w, md, p, st, ms, ma);
  if (a->gate || a->residual || a->slope || a->act) return launch_dense<false, false, kEpiLinearWide>(x, w, md, p, st, ms, ma);
  return launch_dense<false, false, kEpiLinear>(x, w, md, p, st);
}

static bool half_ok(int32_t half, int64_t rows) { return half % 8 == 0 && half >= rows && half <= METIS_TWO_PART_ROWS; }

constexpr int kPointwiseGroups = 64;
extern "C" int64_t metis_linear_pointwise_workspace_bytes(int64_t M, int64_t N) {
  if (M <= 0 || N <= 0) return 0;
  return kPointwiseGroups * N * (int64_t)sizeof(float);
}

static int32_t launch_pointwise(const metis_linear_pointwise_args* a, bool wide, dim3 grid, float* sums) {
  auto launch = [&](auto kern) {
    return launch_counted(kLaunchStream, kern, grid, dim3(256), 0, reinterpret_cast<cudaStream_t>(a->stream),
                             static_cast<const __nv_bfloat16*>(a->dy), a->lddy, static_cast<const __half*>(a->slope), a->ldslope,
                             static_cast<const __nv_bfloat16*>(a->act), a->ldact,
                             static_cast<const __nv_bfloat16*>(a->gate), a->ldgate, a->M, a->N, static_cast<__nv_bfloat16*>(a->dz), a->lddz,
                             (int64_t)(a->dz ? a->half : 0), static_cast<__nv_bfloat16*>(a->dgate), a->lddg, sums);
  };
  METIS_CUDA_OK(wide ? launch(linear_pointwise_kernel<true>) : launch(linear_pointwise_kernel<false>));
  return METIS_OK;
}

extern "C" int32_t metis_linear_pointwise(const metis_linear_pointwise_args* a) {
  if (!a) return fail(METIS_ERR_BAD_ARGUMENT, "args is null");
  if (int32_t rc = check_extent(a->M, "M")) return rc;
  if (int32_t rc = check_extent(a->N, "N")) return rc;
  if (!a->dy || (!a->dz && !a->dgate && !a->dbias)) return fail(METIS_ERR_BAD_ARGUMENT, "dy is null, or nothing is asked for");
  if (a->dgate && !a->act) return fail(METIS_ERR_BAD_ARGUMENT, "act is null");
  if (a->act) if (int32_t rc = check_rows(a->act, a->ldact, a->N, "act")) return rc;
  if (a->slope) if (int32_t rc = check_rows(a->slope, a->ldslope, a->N, "slope")) return rc;
  if (a->dbias && a->dbias_dtype != METIS_DTYPE_BF16 && a->dbias_dtype != METIS_DTYPE_F32) return fail(METIS_ERR_BAD_ARGUMENT, "unknown dbias_dtype %d", a->dbias_dtype);
  if (a->lddy < a->N || (a->gate && a->ldgate < a->N) || (a->dz && a->lddz < a->N) || (a->dgate && a->lddg < a->N))
    return fail(METIS_ERR_BAD_ARGUMENT, "a leading dimension is smaller than N = %lld", (long long)a->N);
  if (a->dbias && (!a->workspace || !aligned16(a->workspace) || a->workspace_bytes < metis_linear_pointwise_workspace_bytes(a->M, a->N)))
    return fail(METIS_ERR_WORKSPACE, "workspace too small or misaligned");
  auto rows16 = [](const void* t, int64_t ld) { return !t || (aligned16(t) && ld % 8 == 0); };
  if (!rows16(a->dz, a->lddz)) return fail(METIS_ERR_BAD_ALIGNMENT, "dz must be 16-byte aligned with a leading dimension that is a multiple of 8");
  for (const void* t : {a->dy, a->gate, static_cast<const void*>(a->dgate)})
    if (reinterpret_cast<uintptr_t>(t) & 1u) return fail(METIS_ERR_BAD_ALIGNMENT, "tensors must be 2-byte aligned");
  const bool wide = a->N % 8 == 0 && rows16(a->dy, a->lddy) && rows16(a->gate, a->ldgate) && rows16(a->dgate, a->lddg);
  if (a->half && !half_ok(a->half, a->M)) return fail(METIS_ERR_BAD_ARGUMENT, "half = %d must be a multiple of 8 from M = %lld to 128", a->half, (long long)a->M);
  const int64_t columns = ceil_div(a->N, 256);
  // with sums no more groups of rows than the workspace has; else about 16 blocks for each SM
  int64_t groups = ceil_div(a->half ? a->half : a->M, 8), most = ceil_div((int64_t)device_sm_count() * 16, columns);
  if (a->dbias && most > kPointwiseGroups) most = kPointwiseGroups;
  if (groups > most) groups = most;
  if (groups > 65535) groups = 65535;
  float* sums = a->dbias ? static_cast<float*>(a->workspace) : nullptr;
  const dim3 grid((unsigned)columns, (unsigned)groups);
  const int32_t rc = launch_pointwise(a, wide, grid, sums);
  if (rc || !a->dbias) return rc;
  const dim3 blocks((unsigned)ceil_div(a->N, 256));
  cudaStream_t st = reinterpret_cast<cudaStream_t>(a->stream);
  if (a->dbias_dtype == METIS_DTYPE_BF16)
    METIS_CUDA_OK(launch_counted(kLaunchShort, linear_bias_kernel<__nv_bfloat16>, blocks, dim3(256), 0, st, (const float*)sums, (int)groups, a->N, static_cast<__nv_bfloat16*>(a->dbias)));
  else
    METIS_CUDA_OK(launch_counted(kLaunchShort, linear_bias_kernel<float>, blocks, dim3(256), 0, st, (const float*)sums, (int)groups, a->N, static_cast<float*>(a->dbias)));
  return METIS_OK;
}

static int32_t finish_sums(const float* sums, const Splits& sp, int64_t M, int64_t N, const int32_t* place_of, int64_t half, const CommonWeight& weight, __nv_bfloat16* d, int64_t ldd, cudaStream_t st) {
  METIS_CUDA_OK(launch_counted(kLaunchStream, finish_sums_kernel, dim3(row_blocks(ceil_div(M * N, 256))), dim3(256), 0, st, sums, (int)sp.splits, sp.rows, M, (int)(N / 8), place_of, half, weight.gout, weight.inv_count, weight.scale, d, ldd));
  return METIS_OK;
}

extern "C" int64_t metis_bf16_product_workspace_bytes(int64_t M, int64_t N, int64_t K, int32_t a_mn_major, int32_t half) {
  if (M <= 0 || N <= 0 || K <= 0 || half < 0) return 0;
  if (half) (a_mn_major ? K : M) = 2 * half;
  SmallShape sh;
  if (!a_mn_major && few_tokens(M, N, K, true, &sh)) return 0;
  const Splits sp = plan_splits(M, N, K);
  return (sp.splits > 1 || (half && !a_mn_major) ? sp.bytes : 0) + (half && a_mn_major ? 4 * (int64_t)half * N : 0);
}

static int32_t stack_rows(const __nv_bfloat16* x, int64_t ldx, int64_t M, int parts, int64_t half, int64_t K, const int64_t* target, int64_t ignore, __nv_bfloat16* out, cudaStream_t st) {
  METIS_CUDA_OK(launch_counted(kLaunchStream, stack_rows_kernel, dim3(row_blocks(ceil_div(parts * half * (K / 8), 32))), dim3(256), 0, st, x, ldx, M, parts, half, K / 8, target, ignore, out));
  return METIS_OK;
}

extern "C" int32_t metis_bf16_product(const void* a, int32_t a_mn_major, int64_t lda, const void* b, int64_t ldb, int64_t M, int64_t N, int64_t K,
                                      int32_t half, void* d, int64_t ldd, void* workspace, int64_t workspace_bytes, int32_t* status, void* stream) {
  if (int32_t rc = check_extent(M, "M")) return rc;
  if (int32_t rc = check_extent(N, "N")) return rc;
  if (int32_t rc = check_extent(K, "K")) return rc;
  if (int32_t rc = check_rows(a, lda, a_mn_major ? M : K, "a")) return rc;
  if (int32_t rc = check_rows(b, ldb, N, "b")) return rc;
  if (int32_t rc = check_rows(d, ldd, N, "d")) return rc;
  if (N % 8 != 0) return fail(METIS_ERR_BAD_SHAPE, "N = %lld must be a multiple of 8", (long long)N);
  if (half && !half_ok(half, a_mn_major ? K : M)) return fail(METIS_ERR_BAD_ARGUMENT, "half = %d must be a multiple of 8 from the rows' number to 128", half);
  const int64_t rows = a_mn_major ? K : M;
  if (half) (a_mn_major ? K : M) = 2 * half;
  SmallShape sh;
  if (!a_mn_major && few_tokens(M, N, K, true, &sh)) {
    DenseParams p = {};
    p.M = M; p.N = N; p.K = K; p.status = status;
    p.half = half; p.half_rows = (int32_t)(half ? rows : 0);
    p.d = static_cast<__nv_bfloat16*>(d); p.ldd = ldd; p.d_wide = 1;
    return launch_dense_small(sh, a, lda, b, true, ldb, p, reinterpret_cast<cudaStream_t>(stream));
  }
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const Splits sp = plan_splits(M, N, K);
  const DenseOperand oa = {a, lda, a_mn_major != 0};
  DenseOperand ob = {b, ldb, true};
  const bool summed = sp.splits > 1 || (half && !a_mn_major);
  const int64_t sum_bytes = summed ? sp.bytes : 0, stack_bytes = half && a_mn_major ? 4 * (int64_t)half * N : 0;
  if (sum_bytes + stack_bytes > 0 && (!workspace || !aligned16(workspace) || workspace_bytes < sum_bytes + stack_bytes))
    return fail(METIS_ERR_WORKSPACE, "workspace too small or misaligned");
  float* sums = static_cast<float*>(workspace);
  if (stack_bytes) {
    __nv_bfloat16* stacked = reinterpret_cast<__nv_bfloat16*>(static_cast<char*>(workspace) + sum_bytes);
    if (int32_t rc = stack_rows(static_cast<const __nv_bfloat16*>(b), ldb, rows, 2, half, N, nullptr, 0, stacked, st)) return rc;
    ob = {stacked, N, true};
  }
  if (!summed) return dense_sum(oa, ob, M, N, K, d, ldd, status, st);
  if (int32_t rc = dense_sum(oa, ob, M, N, K, nullptr, 0, status, st, nullptr, &sp, sums)) return rc;
  return finish_sums(sums, sp, a_mn_major ? M : rows, N, nullptr, a_mn_major ? 0 : half, {}, static_cast<__nv_bfloat16*>(d), ldd, st);
}

// ---- head ---------------------------------------------------------------------------------------------------------

static int32_t check_head(const metis_head_args* a) {
  if (!a) return fail(METIS_ERR_BAD_ARGUMENT, "args is null");
  if (int32_t rc = check_extent(a->M, "M")) return rc;
  if (int32_t rc = check_extent(a->V, "V")) return rc;
  if (int32_t rc = check_extent(a->K, "K")) return rc;
  if (a->K % 8 != 0) return fail(METIS_ERR_BAD_SHAPE, "K = %lld must be a multiple of 8", (long long)a->K);
  if (int32_t rc = check_rows(a->h, a->ldh, a->K, "h")) return rc;
  if (int32_t rc = check_rows(a->w, a->ldw, a->K, "w")) return rc;
  if (a->negate != 0 && a->negate != 1) return fail(METIS_ERR_BAD_ARGUMENT, "negate must be 0 or 1");
  if (!a->target || !a->lse) return fail(METIS_ERR_BAD_ARGUMENT, "target or lse is null");
  if (!(a->scale > 0.0f && a->scale <= 0x1p127f)) return fail(METIS_ERR_BAD_ARGUMENT, "scale = %g must be positive, and at most 2^127: 1.44 times it is finite", (double)a->scale);
  return METIS_OK;
}
constexpr int64_t kFewRows = 64;                           // rows of a head that the weight's read bounds
static int64_t head_slots(int64_t M, int64_t V) { return M <= kFewRows ? small_stats_slots(V) : 2 * ceil_div(V, 256); }

// Packing the rows that are not ignored takes 6 us and the time of two passes over h, on either side, whether there are any or none; from
// 10^12 operations of one product on (0.7 ms) that is 1 to 2 % of the call.  (The threshold is for batches where nothing is ignored.  Where a
// tenth of the rows is, 2048 of them over 151936 x 1536, just below it, would gain 0.3 ms of 3 by it.)
constexpr double kPackFlops = 1e12;
struct HeadPack {
  bool on;
  int32_t *live, *row_of, *place_of;
  __nv_bfloat16* h;
  int64_t bytes;
};
static HeadPack head_pack(int64_t M, int64_t V, int64_t K, void* at) {
  HeadPack k = {};
  k.on = 2.0 * (double)M * (double)V * (double)K >= kPackFlops && M > kFewRows;
  if (!k.on) return k;
  const int64_t index = ceil_div(M * 4, 256) * 256;
  char* b = static_cast<char*>(at);
  k.live = reinterpret_cast<int32_t*>(b);
  k.row_of = reinterpret_cast<int32_t*>(b + 256);
  k.place_of = reinterpret_cast<int32_t*>(b + 256 + index);
  k.h = reinterpret_cast<__nv_bfloat16*>(b + 256 + 2 * index);
  k.bytes = 256 + 2 * index + ceil_div(2 * M * K, 256) * 256;
  return k;
}
static DenseParams head_params(const metis_head_args* a, const HeadPack& pack) {
  DenseParams p = {};
  if (pack.on) { p.row_of = pack.row_of; p.live = pack.live; }
  p.M = a->M; p.N = a->V; p.K = a->K; p.status = a->status;
  p.target = a->target; p.ignore = a->ignore_index; p.vocab = a->V;
  p.weight_scale = a->negate ? -a->scale : a->scale;
  p.scale = a->scale; p.scale_log2e = a->scale * 1.4426950408889634f;
  return p;
}
static int32_t pack_rows(const metis_head_args* a, const HeadPack& k, float* nll, float* entropy, cudaStream_t st) {
  METIS_CUDA_OK(launch_counted(kLaunchShort, head_index_kernel, dim3(1), dim3(1024), 0, st, a->target, a->ignore_index, a->M, k.row_of, k.place_of, k.live, nll, entropy));
  METIS_CUDA_OK(launch_counted(kLaunchStream, head_gather_kernel, dim3(row_blocks(a->M)), dim3(256), 0, st, static_cast<const __nv_bfloat16*>(a->h), a->ldh, a->M,
                                  (int)(a->K / 8), (const int32_t*)k.row_of, (const int32_t*)k.live, k.h));
  return METIS_OK;
}

extern "C" int64_t metis_head_loss_workspace_bytes(int64_t M, int64_t V, int64_t K, int32_t entropy) {
  if (M <= 0 || V <= 0 || K <= 0) return 0;
  return head_pack(M, V, K, nullptr).bytes + head_slots(M, V) * M * (entropy ? 12 : 8);
}

extern "C" int32_t metis_head_loss(const metis_head_args* a, float* nll, float* entropy) { return metis_head_loss_keep(a, nll, entropy, nullptr); }

extern "C" int32_t metis_head_loss_keep(const metis_head_args* a, float* nll, float* entropy, float* target_logp) {
  if (int32_t rc = check_head(a)) return rc;
  if (!nll) return fail(METIS_ERR_BAD_ARGUMENT, "nll is null");
  if (!a->workspace || !aligned16(a->workspace) || a->workspace_bytes < metis_head_loss_workspace_bytes(a->M, a->V, a->K, entropy != nullptr))
    return fail(METIS_ERR_WORKSPACE, "workspace too small or misaligned");
  cudaStream_t st = reinterpret_cast<cudaStream_t>(a->stream);
  const HeadPack pack = head_pack(a->M, a->V, a->K, a->workspace);
  DenseParams p = head_params(a, pack);
  const int64_t slots = head_slots(a->M, a->V);
  p.stats = reinterpret_cast<float2*>(static_cast<char*>(a->workspace) + pack.bytes);
  p.stats_e = entropy ? reinterpret_cast<float*>(p.stats + slots * a->M) : nullptr;
  p.stats_ld = a->M;
  if (pack.on) if (int32_t rc = pack_rows(a, pack, nll, entropy, st)) return rc;
  const DenseOperand h = {pack.on ? pack.h : a->h, pack.on ? a->K : a->ldh, false}, w = {a->w, a->ldw, false};
  const CUtensorMap none = {};
  if (a->M <= kFewRows) {
    if (int32_t rc = launch_dense_small_stats(a->h, a->ldh, a->w, a->ldw, p, st)) return rc;
  } else if (int32_t rc = entropy ? launch_dense<false, false, kEpiStatsEntropy>(h, w, none, p, st) : launch_dense<false, false, kEpiStats>(h, w, none, p, st)) return rc;
  HeadRows r = {};
  r.stats = p.stats; r.stats_e = p.stats_e;
  r.h = static_cast<const __nv_bfloat16*>(h.p); r.ldh = h.ld; r.w = static_cast<const __nv_bfloat16*>(a->w); r.ldw = a->ldw;
  r.target = a->target; r.ignore = a->ignore_index; r.vocab = a->V; r.M = a->M; r.row_of = p.row_of; r.live = p.live;
  r.pieces = (int32_t)(a->K / 8); r.slots = (int32_t)slots;
  r.scale = p.scale; r.scale_log2e = p.scale_log2e; r.sign = a->negate ? -1.0f : 1.0f;
  r.nll = nll; r.lse = a->lse; r.entropy = entropy; r.target_logp = target_logp;
  const bool few = a->M <= kFewRows;
  auto rows = few ? (entropy ? head_rows_kernel<true, 1> : head_rows_kernel<false, 1>) : (entropy ? head_rows_kernel<true, 32> : head_rows_kernel<false, 32>);
  METIS_CUDA_OK(launch_counted(kLaunchShort, rows, dim3((unsigned)ceil_div(a->M, few ? 1 : 32)), dim3(few ? 256 : 1024), 0, st, r));
  return METIS_OK;
}

extern "C" int32_t metis_head_sum(const float* nll, const int64_t* target, int64_t ignore_index, int64_t M, int32_t mean, float* loss, float* inv_count, void* stream) {
  if (int32_t rc = check_extent(M, "M")) return rc;
  if (!nll || !target || !loss || !inv_count) return fail(METIS_ERR_BAD_ARGUMENT, "null pointer");
  METIS_CUDA_OK(launch_counted(kLaunchShort, head_sum_kernel, dim3(1), dim3(1024), 0, reinterpret_cast<cudaStream_t>(stream), nll, target, ignore_index, M, (int)(mean != 0), loss, inv_count));
  return METIS_OK;
}

// What the backward pass keeps: packed rows, the gradients G of a piece's logits, and the sums of dh over pieces and splits (none where one
// product makes it in its place).
struct HeadBackward {
  HeadPack pack;
  int64_t columns;
  Splits sp;
  __nv_bfloat16 *g, *stacked;                              // stacked: h as dw contracts it with G, twice for two parts
  float* sums;
  float* target_logp;                                      // where the call brings none
  int64_t half;                                            // rows from one part of G to the other; 0: it has one
  int64_t bytes;
};

static HeadBackward plan_head_backward(int64_t M, int64_t V, int64_t K, void* at) {
  HeadBackward b = {};
  b.pack = head_pack(M, V, K, at);
  b.half = M <= METIS_TWO_PART_ROWS && !b.pack.on ? ceil_div(M, 8) * 8 : 0;      // G in two parts, see metis_bf16_product
  const int64_t rows = b.half ? 2 * b.half : M;
  b.columns = piece_columns(rows, V);
  b.sp = plan_splits(rows, K, b.columns < V ? b.columns : V);
  const bool summed = b.half || b.pack.on || b.columns < V || b.sp.splits > 1;
  const int64_t g_bytes = ceil_div(2 * rows * b.columns, 256) * 256, sum_bytes = summed ? ceil_div(b.sp.bytes, 256) * 256 : 0;
  b.g = reinterpret_cast<__nv_bfloat16*>(static_cast<char*>(at) + b.pack.bytes);
  b.sums = summed ? reinterpret_cast<float*>(reinterpret_cast<char*>(b.g) + g_bytes) : nullptr;
  b.stacked = reinterpret_cast<__nv_bfloat16*>(reinterpret_cast<char*>(b.g) + g_bytes + sum_bytes);
  const int64_t stacked_bytes = b.pack.on ? 0 : 2 * rows * K;
  b.target_logp = reinterpret_cast<float*>(reinterpret_cast<char*>(b.stacked) + stacked_bytes);
  b.bytes = b.pack.bytes + g_bytes + sum_bytes + stacked_bytes + 4 * M;
  return b;
}

extern "C" int64_t metis_head_backward_workspace_bytes(int64_t M, int64_t V, int64_t K) {
  if (M <= 0 || V <= 0 || K <= 0) return 0;
  return plan_head_backward(M, V, K, nullptr).bytes;
}

extern "C" int32_t metis_head_backward(const metis_head_args* a, const float* gout, int32_t gout_stride, const float* inv_count,
                                       void* dh, int64_t lddh, void* dw, int64_t lddw) {
  return metis_head_backward_kept(a, nullptr, gout, gout_stride, inv_count, dh, lddh, dw, lddw);
}

extern "C" int32_t metis_head_backward_kept(const metis_head_args* a, const float* target_logp, const float* gout, int32_t gout_stride, const float* inv_count,
                                            void* dh, int64_t lddh, void* dw, int64_t lddw) {
  if (int32_t rc = check_head(a)) return rc;
  if (!gout || (!dh && !dw)) return fail(METIS_ERR_BAD_ARGUMENT, "gout is null, or nothing is asked for");
  if (gout_stride && inv_count) return fail(METIS_ERR_BAD_ARGUMENT, "inv_count belongs to one gradient for all rows");
  if (gout_stride != 0 && gout_stride != 1) return fail(METIS_ERR_BAD_ARGUMENT, "gout_stride must be 0 or 1");
  if (dh) if (int32_t rc = check_rows(dh, lddh, a->K, "dh")) return rc;
  if (dw) if (int32_t rc = check_rows(dw, lddw, a->K, "dw")) return rc;
  if (!a->workspace || !aligned16(a->workspace) || a->workspace_bytes < metis_head_backward_workspace_bytes(a->M, a->V, a->K))
    return fail(METIS_ERR_WORKSPACE, "workspace too small or misaligned");
  cudaStream_t st = reinterpret_cast<cudaStream_t>(a->stream);
  const HeadBackward b = plan_head_backward(a->M, a->V, a->K, a->workspace);
  const HeadPack& pack = b.pack;
  const __nv_bfloat16* w = static_cast<const __nv_bfloat16*>(a->w);
  if (pack.on) if (int32_t rc = pack_rows(a, pack, nullptr, nullptr, st)) return rc;
  const DenseOperand h = {pack.on ? pack.h : a->h, pack.on ? a->K : a->ldh, false};
  DenseParams p = head_params(a, pack);
  p.lse = a->lse; p.gout = gout; p.gout_stride = gout_stride;
  p.half = (int32_t)b.half;
  p.target_logp = target_logp ? target_logp : b.target_logp;
  if (!target_logp)
    METIS_CUDA_OK(launch_counted(kLaunchStream, head_target_kernel, dim3(row_blocks(a->M)), dim3(256), 0, st, static_cast<const __nv_bfloat16*>(a->h), a->ldh, w, a->ldw, a->target,
                                 a->ignore_index, a->V, a->M, (int)(a->K / 8), a->scale, (const float*)a->lse, b.target_logp));
  const int64_t rows = b.half ? 2 * b.half : a->M;         // of G
  const DenseOperand of_dw = {pack.on ? pack.h : b.stacked, a->K, true};
  if (!pack.on && dw)
    if (int32_t rc = stack_rows(static_cast<const __nv_bfloat16*>(a->h), a->ldh, a->M, b.half ? 2 : 1, b.half ? b.half : a->M, a->K, a->target, a->ignore_index, b.stacked, st)) return rc;
  const CommonWeight weight = gout_stride ? CommonWeight{} : CommonWeight{gout, inv_count, a->scale};
  for (int64_t v0 = 0; v0 < a->V; v0 += b.columns) {
    const int64_t n = a->V - v0 < b.columns ? a->V - v0 : b.columns;
    CUtensorMap mg = {}, ml = {};
    p.N = n;
    p.col0 = v0;
    if (int32_t rc = map_bf16(&mg, b.g, b.columns, b.half ? b.half : a->M, n, "G")) return rc;
    if (b.half) if (int32_t rc = map_bf16(&ml, b.g + b.half * b.columns, b.columns, b.half, n, "G")) return rc;
    if (int32_t rc = launch_dense<false, false, kEpiGrad>(h, {w + v0 * a->ldw, a->ldw, false}, mg, p, st, ml)) return rc;
    if (dw) {
      if (int32_t rc = dense_sum({b.g, b.columns, true}, of_dw, n, a->K, rows, static_cast<__nv_bfloat16*>(dw) + v0 * lddw, lddw, a->status, st, p.live,
                                 nullptr, nullptr, false, weight)) return rc;
    }
    if (dh) {
      // a shorter last piece has no more splits than the others; those that it leaves out keep what they hold
      const int64_t stages = ceil_div(n, 64);
      Splits sp = b.sp;
      sp.splits = (int32_t)ceil_div(stages, sp.iters_per_split);
      if (int32_t rc = dense_sum({b.g, b.columns, false}, {w + v0 * a->ldw, a->ldw, true}, rows, a->K, n, b.sums ? nullptr : dh, lddh, a->status, st, p.live, &sp, b.sums, v0 > 0, weight)) return rc;
    }
  }
  if (dh && b.sums) return finish_sums(b.sums, b.sp, a->M, a->K, pack.on ? pack.place_of : nullptr, b.half, weight, static_cast<__nv_bfloat16*>(dh), lddh, st);
  return METIS_OK;
}
