// Attention of one new token for each row over a paged key-value cache, split over the keys of all rows and joined.
//
//   s_j = scale q . k_j,   o = sum_j exp(s_j - m) v_j / sum_j exp(s_j - m),   m = max_j s_j
//
// Every key and value is read once and meets the few query heads of its key-value head (6 or 7 in this repository's decoders): 14 flops for each
// byte, which memory bounds as long as the tensor core does them (fp32 units alone would take as long as the memory).  Tiles are of 16 keys.  The keys
// are the rows of the matrix product and the query heads its columns, S^T = K Q^T and O^T = V^T P^T: eight columns hold a whole group, where the
// usual orientation would pad the group to 16 rows and do twice the work; and mma.sync it is, because a tile of 128 rows has nothing to
// put into the other columns that a tcgen05 product would have.
//
// A warp owns its tiles: it brings them by asynchronous copies into its own ring of shared memory (no barrier with other warps), keeps its own running
// maximum, sum and output in registers, and the warps of a block are joined when their row ends.  The flattened list of all tiles of all (row, key-value
// head) pairs is cut into equal parts, one for each block that the GPU holds at once, whatever the lengths are (they are on the device): a block
// finds its part by the sum of the lengths.  A pair that one block covers is finished there; of one that several cover, each writes its maximum, sum
// and output to the workspace, and a second launch joins them in order.
//
// p goes into its product as two bf16 numbers (off by 2^-15 together: the first is less than 2^-7 of p below it, the second rounds that by 2^-8 of
// itself), or with e4m3 one fp16 number, of 2^11 to 2^15 times what it is to the warp's largest: off by 2^-12 of itself, or, below 2^-25 of that one, where it is subnormal,
// by 2^-36 of it (taken as it is, a row with 95 % of its weight on one token lost the others' bits: 2^-25, and all of what lay below).  The rounding of the
// output, 2^-9 on the average, is the only one that counts.  Statistics and sums are fp32.
#include "rollout.cuh"

#include <cuda_fp16.h>
#include <math_constants.h>

namespace metis {
namespace {

constexpr int kRows = 16;                 // keys of one product, which lie on one page
constexpr int kWarps = 4;
constexpr int kThreads = kWarps * 32;
constexpr int kMaxRows = 512;             // of one launch: their sequences and lengths are kept in shared memory
constexpr int kMaxGroup = 1024;           // query heads of a key-value head: their chunks are far fewer than the blocks of a launch
constexpr int64_t kMaxTiles = (int64_t)1 << 30;      // of one launch and one head
constexpr int kMinTiles = 8;              // of a part: two for each warp
// What beginning and ending a row costs a block, in tiles: parts are equal in tiles and this for each row.  A batch of 256 rows of 1 to 2047 keys took
// 85 us where short rows were counted by their tiles alone, 75 with 4, 57 with 16, 56 with 20 to 32; few long rows do not change.
constexpr int kBegin = 20;
constexpr int kUnitThreads = 512;         // of a block that joins one column of many pieces (111 of them: 20.5 us for the call, 20.7 with 256 threads, 21.8 with 1024)
// The maximum of no scores: the lowest finite number, so that a score of -inf weighs nothing behind it, and any other something.  Keys that all score -inf leave it, and 0 / 0; of
// no keys at all (their pages are absent) the maximum is -inf, and the row is zeros.
constexpr float kNone = -3.4028235e38f;
// Weights are relative to a number that is moved when one of them would pass 2^slack: to the largest score, so that bf16 weights are 1 then, or as far under it as fp16, whose smallest
// normal number is 2^-14, is better filled from above.
template <bool kE4m3> constexpr float kSlack = kE4m3 ? 15.0f : 8.0f;
template <bool kE4m3> constexpr float kUnder = kE4m3 ? 11.0f : 0.0f;

struct AttendParams {
  const __nv_bfloat16* q;
  int64_t q_row, q_head;
  __nv_bfloat16* out;
  float* lse;
  const void* slots;
  bool slots_64;
  int32_t rows, heads_q, group, chunks;   // chunks: pieces of a group that a block takes at once
  const int32_t* lengths;
  const int32_t* tables;
  int64_t sequences, width, pages, page_bytes;
  int32_t kv_heads, page_size, head_dim;
  const char* keys;                       // of the layer, on page 0
  int64_t values_off;                     // bytes from keys to values
  const float* scales;                    // [2, kv_heads], or null
  float scale;                            // times log2(e)
  float* part_o;                          // [2 blocks, 8 NT, D]
  float2* part_ml;                        // [2 blocks, 8 NT]
  // What the second launch joins: row, key-value head and chunk as one number, first and last part.  One place for each of those of each row where they are few (by_unit),
  // else one for each block that goes on with what another one began.
  int4* join;
  bool by_unit;
};

__device__ __forceinline__ uint32_t smem_address(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
// 16 bytes, or zeros where `bytes` is 0 (the source is not read then)
__device__ __forceinline__ void copy16(uint32_t to, const void* from, int bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" :: "r"(to), "l"(from), "r"(bytes) : "memory");
}
__device__ __forceinline__ void copy8(uint32_t to, const void* from, int bytes) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 8, %2;" :: "r"(to), "l"(from), "r"(bytes) : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_group %0;" :: "n"(N) : "memory"); }
__device__ __forceinline__ void matrices(uint32_t at, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}
__device__ __forceinline__ void matrices_transposed(uint32_t at, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}
__device__ __forceinline__ uint32_t transpose8(uint32_t v) {
  uint32_t d;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(v));
  return d;
}
template <bool kHalf>
__device__ __forceinline__ void multiply(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (kHalf)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// two e4m3 -> two fp16, exactly
__device__ __forceinline__ uint32_t widen(uint32_t two) {
  uint32_t d;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(d) : "h"((uint16_t)two));
  return d;
}
__device__ __forceinline__ uint32_t bits(__nv_bfloat162 v) { return *reinterpret_cast<uint32_t*>(&v); }
__device__ __forceinline__ uint32_t bits(__half2 v) { return *reinterpret_cast<uint32_t*>(&v); }

// Rows of a tile in shared memory: 16-byte pieces exchanged by the row, so that eight rows' pieces of one column lie in eight different
// groups of banks (rows of 64 bytes lie two to a line of 128).  A lane's row and the low bit of its piece are fixed and the even rest is a constant of
// the unrolled loop, which comes in by one exclusive or.
template <int kRowBytes> __device__ __forceinline__ uint32_t piece_base(int row, int piece) {
  if constexpr (kRowBytes == 64) return row * 64 + (((piece ^ (row >> 1)) & 3) << 4);
  else return row * kRowBytes + ((piece & ~7) << 4) + (((piece ^ row) & 7) << 4);
}
template <int kRowBytes> __device__ __forceinline__ uint32_t piece_next(uint32_t base, int even) {
  constexpr int kMask = kRowBytes == 64 ? 3 : 7;
  return (base ^ ((even & kMask) << 4)) + ((even & ~kMask) << 4);
}

template <int D, int NT, bool kE4m3> struct Plan {
  static constexpr int kItem = kE4m3 ? 1 : 2;
  static constexpr int kRowBytes = D * kItem;
  static constexpr int kPartBytes = kRows * kRowBytes;                  // keys, or values, of 16 tokens
  static constexpr int MT = kE4m3 ? 2 : 1;                              // times 16 keys in a tile: 8-bit ones bring half the bytes for the same softmax
  static constexpr int kTile = kRows * MT;
  static constexpr int kTileBytes = 2 * MT * kPartBytes;
  // Two tiles in the ring: one is worked on while the other comes.  Three blocks of an SM have 12 of them on their way, 96 KB, more than the latency of
  // the memory at its full rate asks for; a third tile would cost one of the blocks.
  static constexpr int kStages = 2;
  static constexpr int kWarpBytes = kStages * kTileBytes;               // >= 8 NT D fp32, which is what a warp leaves there at the end of a row
  static constexpr int kSmem = kWarps * kWarpBytes;
  static constexpr int kPieces = kRowBytes / 16;
  static constexpr int kHeld = D / 16 * NT * 6;                         // registers of output and queries
  static constexpr int kBlocks = kHeld <= 48 ? 3 : 2;
  static_assert(8 * NT * D * 4 <= kWarpBytes, "a warp's output goes where its tiles were");
};

template <int D, int NT, bool kE4m3>
__global__ void __launch_bounds__(kThreads, Plan<D, NT, kE4m3>::kBlocks) attend_kernel(const AttendParams p) {
  using L = Plan<D, NT, kE4m3>;
  constexpr int MT = L::MT;
  extern __shared__ __align__(128) char ring[];
  __shared__ int32_t before[kMaxRows + 1];           // cost of the rows in front, for one key-value head: kBegin and their tiles
  __shared__ int32_t slot_of[kMaxRows], length_of[kMaxRows];
  __shared__ int32_t warp_sums[kWarps];
  __shared__ float2 warp_ml[kWarps][8 * NT];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  grid_dependency_wait();

  // ---- this block's part of the tiles ----
  for (int base = 0; base < p.rows; base += kThreads) {
    const int row = base + threadIdx.x;
    int32_t length = 0;
    if (row < p.rows) {
      const int64_t slot = p.slots ? load_index(p.slots, p.slots_64, row) : row;
      const bool known = slot >= 0 && slot < p.sequences;
      if (known) length = min(max(p.lengths[slot], 0), (int32_t)(p.width * p.page_size));
      slot_of[row] = known ? (int32_t)slot : -1;
      length_of[row] = length;
    }
    const int32_t ahead = base ? before[base] : 0;
    const Scan<int32_t> s = block_scan<kThreads>(length ? (length - 1) / L::kTile + 1 + kBegin : 0, warp_sums);
    if (row <= p.rows) before[row] = ahead + s.before;
    if (threadIdx.x == kThreads - 1 && row < p.rows) before[row + 1] = ahead + s.upto;
    __syncthreads();
  }
  // blocks of the same part are neighbours, one for each chunk of its groups: they read the same tiles at about the same time, and memory once
  // (80 heads on one, 32 rows of 20000 keys: 246 us where each chunk was work of its own, 154 so; 64 on 2: 205 and 128)
  const int heads = p.kv_heads, chunk = blockIdx.x % p.chunks;
  const int64_t total = (int64_t)before[p.rows] * heads;
  const int64_t parts = min((int64_t)(gridDim.x / p.chunks), (total + kMinTiles - 1) / kMinTiles);
  const int64_t cta = blockIdx.x / p.chunks;
  // rows without keys
  for (int row = blockIdx.x; row < p.rows; row += gridDim.x) {
    if (before[row + 1] != before[row]) continue;
    for (int i = threadIdx.x; i < p.heads_q * p.head_dim; i += kThreads) p.out[(int64_t)row * p.heads_q * p.head_dim + i] = __float2bfloat16_rn(0.0f);
    if (p.lse) for (int i = threadIdx.x; i < p.heads_q; i += kThreads) p.lse[(int64_t)row * p.heads_q + i] = -CUDART_INF_F;
    if (p.by_unit) for (int i = threadIdx.x; i < heads * p.chunks; i += kThreads) p.join[row * heads * p.chunks + i] = make_int4(-1, 0, 0, 0);
  }
  if (!p.by_unit && threadIdx.x == 0) p.join[blockIdx.x] = make_int4(-1, 0, 0, 0);
  if (cta >= parts) return;
  int64_t at = cta * total / parts;
  const int64_t end = (cta + 1) * total / parts;

  char* const mine = ring + warp * L::kWarpBytes;
  const uint32_t mine_at = smem_address(mine);
  while (at < end) {
    // the row that the tile belongs to: the last one that begins at or before it (rows without tiles begin where the next one does)
    int lo = 0, hi = p.rows;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if ((int64_t)before[mid] * heads <= at) lo = mid; else hi = mid;
    }
    const int row = lo;
    const int row_cost = before[row + 1] - before[row], row_tiles = row_cost - kBegin;
    const int64_t inside = at - (int64_t)before[row] * heads;
    const int head = (int)(inside / row_cost);
    // this block's tiles of the row and head; their first kBegin places stand for none
    const int here = (int)(inside - (int64_t)head * row_cost);
    const int begin = max(here - kBegin, 0), stop = (int)min((int64_t)row_tiles, here - kBegin + (end - at));
    at += stop > begin ? stop + kBegin - here : end - at;
    if (stop <= begin) continue;           // (the part ends before their first tile)
    const int64_t slot = slot_of[row];
    const int first_head = head * p.group + chunk * 8 * NT, live = min(8 * NT, p.group - chunk * 8 * NT);
    const float k_scale = p.scales ? p.scales[head] : 1.0f, v_scale = p.scales ? p.scales[p.kv_heads + head] : 1.0f;

    // ---- the warp's tiles: begin + warp, and every fourth from there ----
    const int first = begin + warp, tiles_end = stop, keys_all = length_of[row];
    const int mine_count = first < tiles_end ? (tiles_end - first + kWarps - 1) / kWarps : 0;
    const int page_rows = p.page_size / kRows;                            // times 16 keys on a page
    const int32_t* table = p.tables + slot * p.width;
    const int row_bytes = p.head_dim * L::kItem;
    const char* const head_keys = p.keys + (int64_t)head * p.page_size * row_bytes;
    const bool exact = p.head_dim == D;
    // copies: lane's row and piece of the first of a part's 512-byte steps (all further ones by constants where the head has D elements)
    constexpr int kStepRows = 32 / L::kPieces;
    const uint32_t copy_base = piece_base<L::kRowBytes>(lane / L::kPieces, lane % L::kPieces);
    const int column = lane % L::kPieces * 16 < row_bytes ? lane % L::kPieces * 16 : -1;             // of a head of other than D elements; -1: behind its last
    const bool whole_pieces = row_bytes % 16 == 0;
    int32_t page = -1, piece_on_page = 0;  // of the lane's 16 keys among the 32 times 16 that are looked up at once
    int fetched = 0;                       // tiles whose copies have been issued
    uint32_t absent = 0;                   // bit i: the 16 keys i before the last fetched ones lie on no page of the pool
    bool any = false;                      // keys that do
    auto fetch = [&]() {
      if (fetched < mine_count) {
        if ((fetched * MT & 31) == 0) {
          const int which = (first + (fetched + lane / MT) * kWarps) * MT + lane % MT;
          const bool in = which < tiles_end * MT && which * kRows < keys_all;          // (a number of tiles behind the last one may be past 32 bits in keys)
          page = in ? table[which / page_rows] : -1;
          piece_on_page = which % page_rows;
        }
#pragma unroll
        for (int part = 0; part < MT; ++part) {
          const int from_lane = (fetched * MT + part) & 31;
          const int32_t pg = __shfl_sync(0xffffffffu, page, from_lane);
          const int at_page = __shfl_sync(0xffffffffu, piece_on_page, from_lane);
          const bool good = pg >= 0 && pg < p.pages;
          absent = absent << 1 | (good ? 0u : 1u);
          any |= good;
          const int keys = good ? min(kRows, keys_all - ((first + fetched * kWarps) * MT + part) * kRows) : 0;
          const char* from = good ? head_keys + (int64_t)pg * p.page_bytes + at_page * (kRows * row_bytes) : p.keys;
          const uint32_t to = mine_at + (uint32_t)(fetched % L::kStages) * L::kTileBytes + part * 2 * L::kPartBytes;
          if (exact && keys == kRows) {
            const char* src = from + lane * 16;
            const char* src_v = src + p.values_off;
#pragma unroll
            for (int i = 0; i < L::kPartBytes / 512; ++i) {
              // (a step's first row is a multiple of the rows of a step: its bits and the lane's do not meet)
              constexpr int kMask = L::kRowBytes == 64 ? 0 : 7;
              const uint32_t dst = to + ((copy_base ^ ((i * kStepRows & kMask) << 4)) + i * 512);
              copy16(dst, src + i * 512, 16);
              copy16(dst + L::kPartBytes, src_v + i * 512, 16);
            }
          } else if (keys == kRows && (!kE4m3 || whole_pieces)) {
            // Heads of other sizes: a lane's column is the same in all steps, with zeros behind the last one.  (32 rows of 17000 keys, 192 elements: 145 -> 133 us,
            // e4m3 117 -> 78, against the way below; of 80, 20000 keys: 140 -> 138 and 100 -> 84.  Rows on 8 bytes, four copies for two, gain nothing by it.)
            const char* src = from + lane / L::kPieces * row_bytes + max(column, 0);
#pragma unroll
            for (int i = 0; i < L::kPartBytes / 512; ++i) {
              constexpr int kMask = L::kRowBytes == 64 ? 0 : 7;
              const uint32_t dst = to + ((copy_base ^ ((i * kStepRows & kMask) << 4)) + i * 512);
              copy16(dst, src, column < 0 ? 0 : 16);
              copy16(dst + L::kPartBytes, src + p.values_off, column < 0 ? 0 : 16);
              src += kStepRows * row_bytes;
            }
          } else {
#pragma unroll 1
            for (int i = 0; i < L::kPartBytes / 512; ++i) {
              const int piece = i * 32 + lane, r = piece / L::kPieces, c = piece % L::kPieces;
              const bool in = r < keys && c * 16 < row_bytes;
              const char* src = from + (in ? r * row_bytes + c * 16 : 0);
              const uint32_t dst = to + piece_base<L::kRowBytes>(r, c);
              if (!kE4m3 || whole_pieces) {
                copy16(dst, src, in ? 16 : 0);
                copy16(dst + L::kPartBytes, src + p.values_off, in ? 16 : 0);
              } else {
                // (rows of an odd number of 8 bytes begin on 8 bytes alone)
                const bool both = in && c * 16 + 8 < row_bytes;
                copy8(dst, src, in ? 8 : 0);
                copy8(dst + 8, src + (both ? 8 : 0), both ? 8 : 0);
                copy8(dst + L::kPartBytes, src + p.values_off, in ? 8 : 0);
                copy8(dst + L::kPartBytes + 8, src + (both ? 8 : 0) + p.values_off, both ? 8 : 0);
              }
            }
          }
        }
        ++fetched;
      }
      copies_commit();
    };
#pragma unroll
    for (int i = 0; i < L::kStages - 1; ++i) fetch();

    // ---- queries (behind the first copies, which take longer) as the columns of a product: of step i, elements 16 i + 2 t and + 8 of head g (e4m3: in the order in which the keys come) ----
    uint32_t q[NT][D / 16][2];
    float q_scale[NT];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const bool there = n * 8 + g < live;
      const __nv_bfloat16* x = p.q + (int64_t)row * p.q_row + (int64_t)(first_head + n * 8 + g) * p.q_head;
      float biggest = 0.0f;
#pragma unroll
      for (int i = 0; i < D / 16; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const int e = i * 16 + (kE4m3 ? 4 * t + 2 * j : 2 * t + 8 * j);
          q[n][i][j] = there && e < p.head_dim ? *reinterpret_cast<const uint32_t*>(x + e) : 0u;
          if constexpr (kE4m3) biggest = fmaxf(biggest, fmaxf(fabsf(bf16_lo(q[n][i][j])), fabsf(bf16_hi(q[n][i][j]))));
        }
      q_scale[n] = 1.0f;
      if constexpr (kE4m3) {
        // fp16 holds a row of bf16 exactly where it is brought to [1, 2) by a power of two; what lies 2^14 below the row's largest element
        // loses bits that are 2^-25 of that one.  (Infinite and NaN rows stay what they are.)
        biggest = fmaxf(biggest, __shfl_xor_sync(0xffffffffu, biggest, 1));
        biggest = fmaxf(biggest, __shfl_xor_sync(0xffffffffu, biggest, 2));
        const int e = min(max((int)((__float_as_uint(biggest) >> 23) & 255u), 2), 252);
        const float down = __uint_as_float((uint32_t)(254 - e) << 23);
#pragma unroll
        for (int i = 0; i < D / 16; ++i)
#pragma unroll
          for (int j = 0; j < 2; ++j) q[n][i][j] = bits(__floats2half2_rn(bf16_lo(q[n][i][j]) * down, bf16_hi(q[n][i][j]) * down));
        q_scale[n] = __uint_as_float((uint32_t)e << 23);
      }
    }
    // what scores of the columns 2 t and 2 t + 1 are multiplied by
    float s_scale[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int j = 0; j < 2; ++j) s_scale[n][j] = p.scale * k_scale * (kE4m3 ? __shfl_sync(0xffffffffu, q_scale[n], (2 * t + j) * 4) : 1.0f);

    float o[NT][D / 16][4], m[NT][2], l[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
      for (int i = 0; i < D / 16; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) o[n][i][j] = 0.0f;
      m[n][0] = m[n][1] = kNone;
      l[n][0] = l[n][1] = 0.0f;
    }

    const uint32_t k_base = piece_base<L::kRowBytes>(lane & 15, lane >> 4);
    const uint32_t v_base = kE4m3 ? k_base : piece_base<L::kRowBytes>((lane & 7) + ((lane >> 4) << 3), (lane >> 3) & 1);
    for (int done = 0; done < mine_count; ++done) {
      __syncwarp();                        // the tile before this one has been read by all lanes
      fetch();
      copies_wait<L::kStages - 1>();
      __syncwarp();                        // every lane's copies of this tile are there
      const uint32_t tile_at = mine_at + (uint32_t)(done % L::kStages) * L::kTileBytes;
      // ---- scores: keys g and g + 8 of each 16, columns 2 t and 2 t + 1 ----
      constexpr int kChains = MT * NT == 1 ? 2 : 1;                       // (a single sum would wait for each of its products)
      float s[MT][NT][4];
#pragma unroll
      for (int u = 0; u < MT; ++u) {
        float sums[kChains][NT][4];
#pragma unroll
        for (int c = 0; c < kChains; ++c)
#pragma unroll
          for (int n = 0; n < NT; ++n) sums[c][n][0] = sums[c][n][1] = sums[c][n][2] = sums[c][n][3] = 0.0f;
        const uint32_t kt = tile_at + u * 2 * L::kPartBytes + k_base;
        if constexpr (!kE4m3) {
#pragma unroll
          for (int i = 0; i < D / 16; ++i) {
            uint32_t a[4];
            matrices(piece_next<L::kRowBytes>(kt, 2 * i), a);
#pragma unroll
            for (int n = 0; n < NT; ++n) multiply<false>(sums[i % kChains][n], a, q[n][i][0], q[n][i][1]);
          }
        } else {
#pragma unroll
          for (int i = 0; i < D / 16; i += 2) {
            uint32_t r[4];
            matrices(piece_next<L::kRowBytes>(kt, i), r);
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              const uint32_t a[4] = {widen(r[2 * j]), widen(r[2 * j + 1]), widen(r[2 * j] >> 16), widen(r[2 * j + 1] >> 16)};
#pragma unroll
              for (int n = 0; n < NT; ++n) multiply<true>(sums[j % kChains][n], a, q[n][i + j][0], q[n][i + j][1]);
            }
          }
        }
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e) s[u][n][e] = (kChains == 2 ? sums[0][n][e] + sums[kChains - 1][n][e] : sums[0][n][e]) * s_scale[n][e & 1];
      }
      // ---- keys behind the last one, and on no page, weigh nothing ----
      const int left = keys_all - (first + done * kWarps) * L::kTile;
      const uint32_t gone = absent >> ((fetched - 1 - done) * MT);
      if (left < L::kTile || (gone & ((1u << MT) - 1u))) {
#pragma unroll
        for (int u = 0; u < MT; ++u) {
          const int live_keys = (gone >> (MT - 1 - u)) & 1u ? 0 : left - u * kRows;
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (g + (e >> 1) * 8 >= live_keys) s[u][n][e] = -CUDART_INF_F;
        }
      }
      // ---- softmax: what weights are relative to moves when one of them would be too large, and the sums with it ----
      bool over = false;
#pragma unroll
      for (int u = 0; u < MT; ++u)
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e) over |= s[u][n][e] - m[n][e & 1] > kSlack<kE4m3>;
      if (__any_sync(0xffffffffu, over)) {
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            float top = -CUDART_INF_F;
#pragma unroll
            for (int u = 0; u < MT; ++u) top = fmaxf(top, fmaxf(s[u][n][j], s[u][n][2 + j]));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 4));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 8));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 16));
            top = fmaxf(m[n][j], top - kUnder<kE4m3>);
            const float keep = exp2_fast(m[n][j] - top);
            m[n][j] = top;
            l[n][j] *= keep;
#pragma unroll
            for (int i = 0; i < D / 16; ++i) {
              o[n][i][j] *= keep;
              o[n][i][2 + j] *= keep;
            }
          }
      }
      // ---- weights, as the columns of the other product ----
#pragma unroll
      for (int u = 0; u < MT; ++u) {
        uint32_t hi[NT][2], lo_[NT][2];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          float pr[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            pr[e] = exp2_fast(s[u][n][e] - m[n][e & 1]);
            l[n][e & 1] += pr[e];
          }
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            if constexpr (kE4m3) {
              hi[n][r] = transpose8(bits(__floats2half2_rn(pr[2 * r], pr[2 * r + 1])));
            } else {
              // the first part is the largest bf16 below p, so that the second one is positive: zero or negative, it would make NaN of an infinite value
              const uint32_t w = __byte_perm(max(__float_as_uint(pr[2 * r]), 1u) - 1u, max(__float_as_uint(pr[2 * r + 1]), 1u) - 1u, 0x7632);
              hi[n][r] = transpose8(w);
              lo_[n][r] = transpose8(bits(__floats2bfloat162_rn(pr[2 * r] - bf16_lo(w), pr[2 * r + 1] - bf16_hi(w))));
            }
          }
        }
        // ---- values ----
        const uint32_t vt = tile_at + (u * 2 + 1) * L::kPartBytes + v_base;
        if constexpr (!kE4m3) {
#pragma unroll
          for (int i = 0; i < D / 16; ++i) {
            uint32_t a[4];
            matrices_transposed(piece_next<L::kRowBytes>(vt, 2 * i), a);
#pragma unroll
            for (int n = 0; n < NT; ++n) {
              multiply<false>(o[n][i], a, hi[n][0], hi[n][1]);
              multiply<false>(o[n][i], a, lo_[n][0], lo_[n][1]);
            }
          }
        } else {
#pragma unroll
          for (int i = 0; i < D / 16; i += 2) {
            uint32_t r[4];                 // pairs of elements 16 i + 2 g of keys 2 t, 2 t + 1 and 8 more; the same of 16 (i + 1)
            matrices_transposed(piece_next<L::kRowBytes>(vt, i), r);
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              const uint32_t x = __byte_perm(r[2 * j], 0, 0x3120), y = __byte_perm(r[2 * j + 1], 0, 0x3120);
              const uint32_t a[4] = {widen(x), widen(x >> 16), widen(y), widen(y >> 16)};
#pragma unroll
              for (int n = 0; n < NT; ++n) multiply<true>(o[n][i + j], a, hi[n][0], hi[n][1]);
            }
          }
        }
      }
    }
    copies_wait<0>();
    __syncwarp();
    // ---- join the warps; element of o[n][i]: c0, c1 of row g, c2, c3 of row g + 8 of the output's 16 i, columns 2 t, 2 t + 1 ----
    float* const left_o = reinterpret_cast<float*>(mine);
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        float sum = l[n][j];
        sum += __shfl_xor_sync(0xffffffffu, sum, 4);
        sum += __shfl_xor_sync(0xffffffffu, sum, 8);
        sum += __shfl_xor_sync(0xffffffffu, sum, 16);
        const int column = n * 8 + 2 * t + j;
        if (g == 0) warp_ml[warp][column] = make_float2(any ? m[n][j] : -CUDART_INF_F, sum);
#pragma unroll
        for (int i = 0; i < D / 16; ++i) {
          const int e0 = i * 16 + (kE4m3 ? 2 * g : g), e1 = i * 16 + (kE4m3 ? 2 * g + 1 : g + 8);
          left_o[column * D + e0] = o[n][i][j];
          left_o[column * D + e1] = o[n][i][2 + j];
        }
      }
    __syncthreads();
    const bool whole = begin == 0 && stop == row_tiles;
    const int64_t place = ((int64_t)blockIdx.x * 2 + (begin == 0 ? 1 : 0)) * 8 * NT;
    for (int i = threadIdx.x; i < live * D; i += kThreads) {
      const int column = i / D, e = i - column * D;
      float top = -CUDART_INF_F;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) top = fmaxf(top, warp_ml[w][column].x);
      const bool none = top == -CUDART_INF_F;
      float sum = 0.0f, acc = 0.0f;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        const float2 ml = warp_ml[w][column];
        const float f = exp2_fast(ml.x - top);
        sum += ml.y * f;
        acc += reinterpret_cast<const float*>(ring + w * L::kWarpBytes)[i] * f;
      }
      if (none) sum = acc = 0.0f;          // (NaN of -inf less -inf)
      if (whole) {
        const int64_t to = (int64_t)row * p.heads_q + first_head + column;
        if (e < p.head_dim) p.out[to * p.head_dim + e] = __float2bfloat16_rn(none ? 0.0f : __fdiv_rn(acc, sum) * v_scale);
        if (e == 0 && p.lse) p.lse[to] = (top + log2f(sum)) * 0.69314718055994531f;
      } else {
        p.part_o[(place + column) * D + e] = acc;
        if (e == 0) p.part_ml[place + column] = make_float2(top, sum);
      }
    }
    if (threadIdx.x == 0 && (p.by_unit ? begin == 0 : begin > 0)) {
      const int64_t start = (int64_t)before[row] * heads + (int64_t)head * row_cost + kBegin, last = start + row_tiles - 1;
      const int unit = head * p.chunks + chunk;
      p.join[p.by_unit ? row * heads * p.chunks + unit : (int)blockIdx.x] =
          make_int4(whole ? -1 : row, unit, (int)(((start + 1) * parts - 1) / total), (int)(((last + 1) * parts - 1) / total));
    }
    __syncthreads();                       // the ring is free again
  }
}

// Joins the pieces of a row and head that several blocks wrote.  A lane has D / 32 elements of one column (query head of the group), a warp some of its pieces, kAhead of them on
// their way at once and the maxima beside them.
//   by_unit   few rows and heads, of many pieces: a block for each column, whose warps share the pieces
//   else      as many blocks as wrote pieces, and all but the first of those of one row and head share its columns among them, and a block's warps their pieces: of two pieces
//             one block joins all columns, a warp each; of 100 a block joins one column with all its warps.  (256 rows in two or three pieces, with the rest of
//             the call: 55.0 us by a block for each column and piece, 52.5 so; one row of 32768 keys 20.5 by unit, 23.6 this way.  64 rows of four
//             pieces 31.1 by unit in blocks of 256 threads, 29.4 so.)
template <int D> struct alignas(D == 64 ? 8 : 16) Lane { float v[D / 32]; };
template <int D, int NT, bool kByUnit, int kJoinThreads>
__global__ void __launch_bounds__(kJoinThreads) join_kernel(const AttendParams p) {
  constexpr int kJoinWarps = kJoinThreads / 32, E = D / 32, kAhead = 4;
  __shared__ Lane<D> acc_of[kJoinWarps][32];
  __shared__ float sum_of[kJoinWarps];
  grid_dependency_wait();
  const int4 job = p.join[blockIdx.x];
  if (job.x < 0) return;
  const int head = job.y / p.chunks, chunk = job.y - head * p.chunks;
  const int columns = min(8 * NT, p.group - chunk * 8 * NT), pieces = job.w - job.z + 1;
  const int helpers = kByUnit ? gridDim.y : pieces - 1, mine = kByUnit ? (int)blockIdx.y : (int)(blockIdx.x / p.chunks) - job.z - 1;        // blocks that share the columns
  const int here = (columns - mine + helpers - 1) / helpers;
  if (here <= 0) return;
  int share = kJoinWarps;                  // warps of a column
  while (share > 1 && share * here > kJoinWarps) share >>= 1;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, first = warp % share;
  const float v_scale = p.scales ? p.scales[p.kv_heads + head] : 1.0f;
  for (int i = warp / share; i - warp / share < here; i += kJoinWarps / share) {
    const int column = mine + i * helpers;
    const bool live = i < here;
    auto place = [&](int piece) { return (((int64_t)(job.z + piece) * p.chunks + chunk) * 2 + (piece == 0 ? 1 : 0)) * 8 * NT + column; };
    Lane<D> acc;
    float sum = 0.0f, top = -CUDART_INF_F;
#pragma unroll
    for (int e = 0; e < E; ++e) acc.v[e] = 0.0f;
    if (live) {
      float2 ml[kAhead];
      Lane<D> o[kAhead];
      auto load = [&](int from) {
#pragma unroll
        for (int a = 0; a < kAhead; ++a) {
          const int64_t at = place(min(from + a * share, pieces - 1));
          ml[a] = p.part_ml[at];
          o[a] = reinterpret_cast<const Lane<D>*>(p.part_o + at * D)[lane];
        }
      };
      load(first);
      for (int j = lane; j < pieces; j += 32) top = fmaxf(top, p.part_ml[place(j)].x);
#pragma unroll
      for (int s = 16; s > 0; s >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, s));
      for (int from = first; from < pieces;) {
#pragma unroll
        for (int a = 0; a < kAhead; ++a) {
          if (from + a * share >= pieces) continue;
          const float f = exp2_fast(ml[a].x - top);
          sum += ml[a].y * f;
#pragma unroll
          for (int e = 0; e < E; ++e) acc.v[e] += o[a].v[e] * f;
        }
        from += kAhead * share;
        if (from < pieces) load(from);
      }
    }
    if (share > 1) {                       // (then there is one round, and all threads are in it)
      acc_of[warp][lane] = acc;
      if (lane == 0) sum_of[warp] = sum;
      __syncthreads();
      if (first > 0) continue;
      for (int w = 1; w < share; ++w) {
        const Lane<D> other = acc_of[warp + w][lane];
        sum += sum_of[warp + w];
#pragma unroll
        for (int e = 0; e < E; ++e) acc.v[e] += other.v[e];
      }
    }
    if (!live) continue;
    const int64_t to = (int64_t)job.x * p.heads_q + head * p.group + chunk * 8 * NT + column;
    const bool none = top == -CUDART_INF_F;
#pragma unroll
    for (int e = 0; e < E; e += 2)
      if (lane * E + e < p.head_dim)
        *reinterpret_cast<__nv_bfloat162*>(p.out + to * p.head_dim + lane * E + e) =
            __floats2bfloat162_rn(none ? 0.0f : __fdiv_rn(acc.v[e], sum) * v_scale, none ? 0.0f : __fdiv_rn(acc.v[e + 1], sum) * v_scale);
    if (lane == 0 && p.lse) p.lse[to] = none ? top : (top + log2f(sum)) * 0.69314718055994531f;
  }
}

// ---- host -----------------------------------------------------------------------------------------------------------

int padded_dim(int head_dim) { return head_dim <= 64 ? 64 : head_dim <= 128 ? 128 : 256; }
// Columns of eight that a block takes at once; of larger groups, 16 heads each, 8 of more than 128 elements.  (Four of them hold 255 registers and one block an
// SM: 256 rows of 1000 keys, 64 heads on 2 of 128 elements, 96.8 us, 98.2 in e4m3, for 88.0 and 77.7; 80 heads on one, 32 rows of 20000 keys, 185 and 151 us for 154
// and 121; of 64 elements, 48 on 2, 72 and 58 for 79 and 64.  Two of 256 elements are one block an SM, too: 40 heads on one, 32 rows of 13000 keys, 205 and 154 us for
// 177 and 137; 24 on 2, 7000 keys, 86.9 and 71.9 for 90.6 and 66.4; one row of 20000, 21.3 and 22.2 for 17.8 and 16.5.)
int column_tiles(int group, int D) { return group <= 8 || D == 256 ? 1 : 2; }

template <int D, int NT, bool kE4m3>
struct Launch {
  using L = Plan<D, NT, kE4m3>;
  static int64_t workspace(int64_t blocks) { return blocks * (16 + 16 * NT * (8 + D * 4)); }
  // as many as the GPU holds at once
  static int32_t blocks(int64_t* n) {
    if (const cudaError_t e = allow_smem<&attend_kernel<D, NT, kE4m3>>(L::kSmem); e != cudaSuccess) return fail(METIS_ERR_CUDA, "paged attention: %s", cudaGetErrorString(e));
    *n = (int64_t)device_sm_count() * resident_ctas(reinterpret_cast<const void*>(attend_kernel<D, NT, kE4m3>), kThreads, L::kSmem);
    return METIS_OK;
  }
  static int32_t run(AttendParams p, void* ws, int64_t ws_bytes, cudaStream_t st) {
    int64_t n = 0;
    if (const int32_t rc = blocks(&n)) return rc;
    if (ws_bytes < workspace(n)) return fail(METIS_ERR_WORKSPACE, "the workspace has %lld bytes, %lld are needed", (long long)ws_bytes, (long long)workspace(n));
    if (p.chunks > n) return fail(METIS_ERR_UNSUPPORTED, "the GPU holds %lld blocks, fewer than the group has pieces (%d)", (long long)n, p.chunks);
    const int64_t units = (int64_t)p.rows * p.kv_heads * p.chunks;
    p.by_unit = units * 8 <= n;
    char* w = static_cast<char*>(ws);
    p.join = reinterpret_cast<int4*>(w);
    p.part_ml = reinterpret_cast<float2*>(w + n * 16);
    p.part_o = reinterpret_cast<float*>(w + n * (16 + 16 * NT * 8));
    METIS_CUDA_OK(launch_overlapped(kLaunchShort, attend_kernel<D, NT, kE4m3>, dim3((unsigned)n), dim3(kThreads), L::kSmem, st, p));
    const int columns = p.group < 8 * NT ? p.group : 8 * NT;
    if (p.by_unit) METIS_CUDA_OK(launch_overlapped(kLaunchShort, join_kernel<D, NT, true, kUnitThreads>, dim3((unsigned)units, (unsigned)columns), dim3(kUnitThreads), 0, st, p));
    else           METIS_CUDA_OK(launch_overlapped(kLaunchShort, join_kernel<D, NT, false, 256>, dim3((unsigned)n), dim3(256), 0, st, p));
    count_rollout_launches(2);
    return METIS_OK;
  }
};

// f(Launch<...>()) of the kernel for these sizes
template <typename F>
int32_t with_kernel(int head_dim, int group, bool e4m3, const F& f) {
  const int D = padded_dim(head_dim), nt = column_tiles(group, D);
  if (D == 64)  return nt == 1 ? (e4m3 ? f(Launch<64, 1, true>()) : f(Launch<64, 1, false>())) : (e4m3 ? f(Launch<64, 2, true>()) : f(Launch<64, 2, false>()));
  if (D == 128) return nt == 1 ? (e4m3 ? f(Launch<128, 1, true>()) : f(Launch<128, 1, false>())) : (e4m3 ? f(Launch<128, 2, true>()) : f(Launch<128, 2, false>()));
  return e4m3 ? f(Launch<256, 1, true>()) : f(Launch<256, 1, false>());
}

}  // namespace
}  // namespace metis

using namespace metis;

extern "C" int64_t metis_cache_attend_workspace_bytes(const metis_cache* c, int64_t rows, int32_t heads_q) {
  if (!c || rows <= 0 || c->kv_heads <= 0 || heads_q <= 0 || c->head_dim <= 0 || c->head_dim > 256) return 0;
  int64_t bytes = 0;
  const int32_t rc = with_kernel(c->head_dim, heads_q / c->kv_heads, c->dtype == METIS_DTYPE_E4M3, [&](auto kernel) {
    int64_t n = 0;
    const int32_t failed = kernel.blocks(&n);
    bytes = kernel.workspace(n);
    return failed;
  });
  return rc ? 0 : bytes;
}

extern "C" int32_t metis_cache_attend(const metis_cache* cache, const metis_attend_args* a) {
  CacheView c;
  if (const int32_t rc = check_cache(cache, &c)) return rc;
  if (!a || !a->q || !a->out || !a->workspace) return fail(METIS_ERR_BAD_ARGUMENT, "null pointer");
  if (a->rows <= 0 || a->heads_q <= 0 || a->heads_q % c.kv_heads != 0 || a->layer < 0 || a->layer >= c.layers)
    return fail(METIS_ERR_BAD_SHAPE, "rows must be positive, heads_q a multiple of kv_heads and the layer one of the cache");
  if (a->q_row % 2 != 0 || a->q_head % 2 != 0 || (reinterpret_cast<uintptr_t>(a->q) & 3) || !aligned16(a->workspace))
    return fail(METIS_ERR_BAD_ALIGNMENT, "rows of q must be 4-byte aligned and the workspace 16");
  const int group = a->heads_q / c.kv_heads, nt = column_tiles(group, padded_dim(c.head_dim));
  if (group > kMaxGroup) return fail(METIS_ERR_TOO_LARGE, "at most %d query heads share a key-value head", kMaxGroup);
  const int64_t part = (int64_t)c.kv_heads * c.page_size * c.head_dim * c.item;
  const cudaStream_t st = static_cast<cudaStream_t>(a->stream);
  // more rows than one launch counts go in several, one after the other: they share the workspace
  const int64_t row_tiles = c.width * c.page_size / kRows, most = kMaxTiles / row_tiles < kMaxRows ? kMaxTiles / row_tiles : kMaxRows;
  for (int64_t row = 0; row < a->rows; row += most) {
    AttendParams p = {};
    p.rows = (int32_t)min(most, a->rows - row);
    p.q = static_cast<const __nv_bfloat16*>(a->q) + row * a->q_row; p.q_row = a->q_row; p.q_head = a->q_head;
    p.out = static_cast<__nv_bfloat16*>(a->out) + row * a->heads_q * c.head_dim;
    p.lse = a->lse ? a->lse + row * a->heads_q : nullptr;
    p.slots = a->slots ? static_cast<const char*>(a->slots) + row * (a->slots_64 ? 8 : 4) : nullptr;
    p.slots_64 = a->slots_64 != 0;
    p.heads_q = a->heads_q; p.group = group; p.chunks = (group + 8 * nt - 1) / (8 * nt);
    p.lengths = c.lengths; p.tables = c.tables; p.sequences = c.sequences; p.width = c.width;
    if (!a->slots && row > 0) {              // row i of the launch is sequence row + i
      p.lengths += row; p.tables += row * c.width; p.sequences = c.sequences > row ? c.sequences - row : 0;
    }
    p.pages = c.pages; p.page_bytes = c.page_bytes; p.kv_heads = c.kv_heads; p.page_size = c.page_size; p.head_dim = c.head_dim;
    p.keys = c.pool + a->layer * 2 * part;
    p.values_off = part;
    p.scales = cache->scales ? cache->scales + (int64_t)a->layer * 2 * c.kv_heads : nullptr;
    p.scale = a->scale * 1.4426950408889634f;
    const int32_t rc = with_kernel(c.head_dim, group, c.item == 1, [&](auto kernel) { return kernel.run(p, a->workspace, a->workspace_bytes, st); });
    if (rc != METIS_OK) return rc;
  }
  return METIS_OK;
}
