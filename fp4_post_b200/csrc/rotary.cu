// Rotary positions, and the same with the keys and values written into a paged cache.
//
// A pair (a, b) of a head at position p goes to m (a cos - b sin, b cos + a sin) of the angle 2 pi p f, f a frequency in turns per position.  f is held
// as a 64-bit fraction of a turn: p f modulo 1 is then one integer product whose high bits are thrown away, exact for the fraction that is given, and the angle never needs a
// range reduction (fp32 products of positions and frequencies are off by p 2^-24, a whole radian at 2^24).  The fractions that rollout.Rotary gives come from the
// host's 64-bit floats: off by up to 2^-53 turns (theta^(-2i / d) and its quotient by 2 pi, a few steps of what is at most 0.16), so that an angle is off by
// p 2^-53 turns: below fp32's own rounding to p = 2^26.
// No table of cosines is kept or read: a block forms those of its tokens once, in shared memory, and uses them for all heads.
//
// Bound by memory: every element is read and written once.  A thread holds the cosines of one unit (16 bytes of each half, or 16 bytes of
// neighbouring pairs) in registers and takes it through the heads of its token; of few tokens, heads are spread over the block instead.  Appending prompts is bound by
// latency: 45 % of the memory's rate and of the issue slots, with 24 warps an SM and a thread's keys and values behind its queries.
#include "rollout.cuh"

#include <type_traits>

namespace metis {
namespace {

constexpr int kThreads = 256;

struct RotaryShape {
  int32_t heads_q, heads_k, head_dim, rotary_dim;
  int32_t units, rotary_units;        // of a head: all, and those that turn
  int32_t head_lanes, block_tokens;   // threads that share a token's heads, tokens that a block takes at once
  int32_t span;                       // and in all, one group of block_tokens after the other
  float magnitude, sign;              // what cosines and sines are multiplied by; the direction
};

template <typename T> struct Vec;
template <> struct Vec<__nv_bfloat16> {
  static constexpr int kWide = 8;
  static __device__ __forceinline__ void unpack(const uint4& w, float (&v)[8]) {
    v[0] = bf16_lo(w.x); v[1] = bf16_hi(w.x); v[2] = bf16_lo(w.y); v[3] = bf16_hi(w.y);
    v[4] = bf16_lo(w.z); v[5] = bf16_hi(w.z); v[6] = bf16_lo(w.w); v[7] = bf16_hi(w.w);
  }
  static __device__ __forceinline__ void store(__nv_bfloat16* p, const float (&v)[8]) {
    uint4 w;
    __nv_bfloat162 t[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) t[i] = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
    w.x = *reinterpret_cast<uint32_t*>(&t[0]); w.y = *reinterpret_cast<uint32_t*>(&t[1]);
    w.z = *reinterpret_cast<uint32_t*>(&t[2]); w.w = *reinterpret_cast<uint32_t*>(&t[3]);
    *reinterpret_cast<uint4*>(p) = w;
  }
  static __device__ __forceinline__ float one(const __nv_bfloat16* p) { return __bfloat162float(*p); }
  static __device__ __forceinline__ void put(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }
};
template <> struct Vec<float> {
  static constexpr int kWide = 4;
  static __device__ __forceinline__ void unpack(const uint4& w, float (&v)[4]) {
    v[0] = __uint_as_float(w.x); v[1] = __uint_as_float(w.y); v[2] = __uint_as_float(w.z); v[3] = __uint_as_float(w.w);
  }
  static __device__ __forceinline__ void store(float* p, const float (&v)[4]) { *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]); }
  static __device__ __forceinline__ float one(const float* p) { return *p; }
  static __device__ __forceinline__ void put(float* p, float v) { *p = v; }
};

// cos and sin of the pair of frequency `turn` at a position.  Whole quarter turns are taken off while the angle is a whole number: what is left, at most an eighth of a turn, keeps
// its own 24 bits in fp32, where the whole angle would be rounded to 2^-25 of half a turn and a sine near zero lose most of its bits.
__device__ __forceinline__ float2 cos_sin(uint64_t turn, int64_t position, const RotaryShape& s) {
  const uint64_t part = turn * (uint64_t)position;
  const uint32_t quarter = (uint32_t)((part + (1ull << 61)) >> 62);
  float sn, cs;
  sincospif((float)(int32_t)((int64_t)(part - ((uint64_t)quarter << 62)) >> 30) * 0x1p-33f, &sn, &cs);
  const float c = (quarter & 1) ? sn : cs, d = (quarter & 1) ? cs : sn;
  return make_float2((((quarter + 1) & 2) ? -c : c) * s.magnitude, ((quarter & 2) ? -d : d) * s.magnitude * s.sign);
}

// A unit of a head: the two pieces of W elements of the half layout, one piece of W elements of neighbouring pairs, with W = 1 the two elements of a
// pair.  What does not turn goes in units of the same kind: two pieces behind one another (the last one twice where there is an odd one) or one.
// Where they are is the same in all heads, and nothing branches: the arrays of a batch have to stay in registers.
template <int W, bool kInterleaved> __host__ __device__ constexpr bool two_pieces() { return W == 1 || !kInterleaved; }
struct Unit {
  int at, bt;
  bool turns;
};
template <int W, bool kInterleaved>
__device__ __forceinline__ Unit unit_of(int unit, const RotaryShape& s) {
  constexpr bool kTwo = two_pieces<W, kInterleaved>();
  if (unit >= s.rotary_units) {
    const int at = s.rotary_dim + (unit - s.rotary_units) * W * (kTwo ? 2 : 1);
    return {at, min(at + W, s.head_dim - W), false};
  }
  if (W == 1 && kInterleaved) return {2 * unit, 2 * unit + 1, true};
  return {unit * W, unit * W + s.rotary_dim / 2, true};
}
template <typename T, int W, bool kTwo>
struct Raw {
  uint4 a, b;
  __device__ __forceinline__ void load(const T* x, const Unit& u) {
    a = *reinterpret_cast<const uint4*>(x + u.at);
    if constexpr (kTwo) b = *reinterpret_cast<const uint4*>(x + u.bt);
  }
};
template <typename T>
struct Raw<T, 1, true> {
  float a, b;
  __device__ __forceinline__ void load(const T* x, const Unit& u) {
    a = Vec<T>::one(x + u.at);
    b = Vec<T>::one(x + u.bt);
  }
};
template <typename T, int W, bool kInterleaved, typename Put>
__device__ __forceinline__ void turn_unit(const Raw<T, W, two_pieces<W, kInterleaved>()>& r, const Unit& at, const float2 (&c)[W], const Put& put) {
  if constexpr (W == 1) {
    put.one(at.at, at.turns ? fmaf(r.a, c[0].x, -r.b * c[0].y) : r.a);
    put.one(at.bt, at.turns ? fmaf(r.b, c[0].x, r.a * c[0].y) : r.b);
  } else {
    float a[W];
    Vec<T>::unpack(r.a, a);
    if constexpr (kInterleaved) {
#pragma unroll
      for (int i = 0; i < W; i += 2) {
        const float u = a[i], v = a[i + 1];
        a[i] = at.turns ? fmaf(u, c[i / 2].x, -v * c[i / 2].y) : u;
        a[i + 1] = at.turns ? fmaf(v, c[i / 2].x, u * c[i / 2].y) : v;
      }
      put.wide(at.at, a);
    } else {
      float b[W];
      Vec<T>::unpack(r.b, b);
#pragma unroll
      for (int i = 0; i < W; ++i) {
        const float u = a[i], v = b[i];
        a[i] = at.turns ? fmaf(u, c[i].x, -v * c[i].y) : u;
        b[i] = at.turns ? fmaf(v, c[i].x, u * c[i].y) : v;
      }
      put.wide(at.at, a);
      put.wide(at.bt, b);
    }
  }
}
// Heads of one token, kPieces pieces read before the first is written (outputs might be inputs, for all that the compiler knows, and each load would
// wait for the store before it).  Behind the last head the last is read again, and not written.  Four pieces and four blocks an SM: 8192 tokens of 28 + 4
// heads 26.2 -> 23.9 us, pairs of neighbours 33.6 -> 26.1; eight and three: 27.3 and 27.1.  Appending, which has keys and values on their way as well, takes eight
// and three (50.4 us for the padded prompts, 52.1 with four).
template <typename T, int W, bool kInterleaved, int kPieces, typename MakePut>
__device__ __forceinline__ void turn_heads(const T* x, int64_t head_stride, int lane, int heads, int lanes, const Unit& at, const float2 (&c)[W], const MakePut& put_of) {
  constexpr bool kTwo = two_pieces<W, kInterleaved>();
  constexpr int kBatch = kTwo ? kPieces / 2 : kPieces;
  for (int h = lane; h < heads; h += kBatch * lanes) {
    Raw<T, W, kTwo> r[kBatch];
#pragma unroll
    for (int i = 0; i < kBatch; ++i) r[i].load(x + min(h + i * lanes, heads - 1) * head_stride, at);
#pragma unroll
    for (int i = 0; i < kBatch; ++i)
      if (h + i * lanes < heads) turn_unit<T, W, kInterleaved>(r[i], at, c, put_of(h + i * lanes));
  }
}

// pairs of a unit
template <int W, bool kInterleaved> __host__ __device__ constexpr int unit_pairs() { return W == 1 ? 1 : kInterleaved ? W / 2 : W; }

// The cosines of this thread's unit, out of the block's table of its tokens.
template <int W, bool kInterleaved>
__device__ __forceinline__ void unit_table(const float2* table, int token, int unit, int pairs, bool turns, float2 (&c)[W]) {
  constexpr int P = unit_pairs<W, kInterleaved>();
#pragma unroll
  for (int i = 0; i < P; ++i) c[i] = turns ? table[token * pairs + unit * P + i] : make_float2(1.0f, 0.0f);
}

template <typename T> struct PutDense {
  T* out;
  __device__ __forceinline__ void one(int i, float v) const { Vec<T>::put(out + i, v); }
  __device__ __forceinline__ void wide(int i, const float (&v)[Vec<T>::kWide]) const { Vec<T>::store(out + i, v); }
};

struct RotaryTensors {
  const void* positions;
  int64_t tokens, inner;
  const uint64_t* turns;
  const void *q, *k;
  int64_t q_outer, q_token, q_head, k_outer, k_token, k_head;
  void *q_out, *k_out;
  bool positions_64;
};

template <typename T, int W, bool kInterleaved>
__global__ void __launch_bounds__(kThreads, 4) rotary_kernel(const RotaryTensors t, const RotaryShape s) {
  extern __shared__ float2 table[];
  grid_dependency_wait();
  const int pairs = s.rotary_dim / 2;
  const int64_t first = (int64_t)blockIdx.x * s.span;
  const int here = (int)min((int64_t)s.span, t.tokens - first);
  for (int i = threadIdx.x; i < here * pairs; i += kThreads) {
    const int token = i / pairs;
    const int64_t at = first + token;
    table[i] = cos_sin(t.turns[i - token * pairs], t.positions ? load_index(t.positions, t.positions_64, at) : at % t.inner, s);
  }
  __syncthreads();
  const int unit = threadIdx.x % s.units, rest = threadIdx.x / s.units;
  const int lane = rest % s.head_lanes;
  const Unit at_unit = unit_of<W, kInterleaved>(unit, s);
  if (rest >= s.head_lanes * s.block_tokens) return;
  for (int token = rest / s.head_lanes; token < here; token += s.block_tokens) {
    float2 c[W];
    unit_table<W, kInterleaved>(table, token, unit, pairs, at_unit.turns, c);
    const int64_t at = first + token, outer = at / t.inner, inner = at - outer * t.inner;
    const T* q = static_cast<const T*>(t.q) + outer * t.q_outer + inner * t.q_token;
    T* q_out = static_cast<T*>(t.q_out) + at * s.heads_q * s.head_dim;
    turn_heads<T, W, kInterleaved, 4>(q, t.q_head, lane, s.heads_q, s.head_lanes, at_unit, c, [&](int h) { return PutDense<T>{q_out + (int64_t)h * s.head_dim}; });
    if (s.heads_k == 0) continue;
    const T* k = static_cast<const T*>(t.k) + outer * t.k_outer + inner * t.k_token;
    T* k_out = static_cast<T*>(t.k_out) + at * s.heads_k * s.head_dim;
    turn_heads<T, W, kInterleaved, 4>(k, t.k_head, lane, s.heads_k, s.head_lanes, at_unit, c, [&](int h) { return PutDense<T>{k_out + (int64_t)h * s.head_dim}; });
  }
}

// ---- append -------------------------------------------------------------------------------------------------------

struct AppendTensors {
  CacheView cache;
  char* layer_pool;                 // the layer's keys on page 0
  const float* scales;              // [2, kv_heads] of the layer, or null
  const void *slots, *positions;
  int64_t tokens;
  const uint64_t* turns;            // null: nothing turns
  const __nv_bfloat16 *q, *k, *v;
  int64_t q_token, q_head, k_token, k_head, v_token, v_head;
  __nv_bfloat16* q_out;
  bool slots_64, positions_64;
};

// Elements of the cache: bf16 as they are, e4m3 as x / scale rounded to nearest and saturated (NaN stays NaN).  The quotient is the IEEE one:
// a product with a reciprocal is off by up to one bit of fp32, which at a border of the format is a step of 2^-3.
template <bool kE4m3> struct PutCache;
template <> struct PutCache<false> {
  __nv_bfloat16* out;
  float scale;
  __device__ __forceinline__ void one(int i, float v) const { out[i] = __float2bfloat16_rn(v); }
  __device__ __forceinline__ void wide(int i, const float (&v)[8]) const { Vec<__nv_bfloat16>::store(out + i, v); }
};
template <> struct PutCache<true> {
  uint8_t* out;
  float scale;
  __device__ __forceinline__ void one(int i, float v) const { out[i] = float_to_e4m3(__fdiv_rn(v, scale)); }
  __device__ __forceinline__ void wide(int i, const float (&v)[8]) const {
    uint32_t w[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(__fdiv_rn(v[4 * j], scale), __fdiv_rn(v[4 * j + 1], scale)), __NV_SATFINITE, __NV_E4M3);
      const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(__fdiv_rn(v[4 * j + 2], scale), __fdiv_rn(v[4 * j + 3], scale)), __NV_SATFINITE, __NV_E4M3);
      w[j] = lo | (hi << 16);
    }
    *reinterpret_cast<uint2*>(out + i) = make_uint2(w[0], w[1]);
  }
};

// One block takes tokens, and the heads of q, k and v of each, as rotary_kernel does.  What a token goes to is looked up once, by one thread.
template <int W, bool kInterleaved, bool kE4m3>
__global__ void __launch_bounds__(kThreads, 3) append_kernel(const AppendTensors t, const RotaryShape s) {
  extern __shared__ float2 table[];
  int64_t* const token_at = reinterpret_cast<int64_t*>(table + s.span * (s.rotary_dim / 2));      // bytes from layer_pool to the token's row in the keys of head 0, -1: nowhere, -2: no sequence
  int64_t* const token_position = token_at + s.span;
  grid_dependency_wait();
  const CacheView& c = t.cache;
  const int pairs = s.rotary_dim / 2;
  const int64_t first = (int64_t)blockIdx.x * s.span;
  const int here = (int)min((int64_t)s.span, t.tokens - first);
  for (int n = threadIdx.x; n < here; n += kThreads) {
    const int64_t i = first + n, slot = t.slots ? load_index(t.slots, t.slots_64, i) : i;
    int64_t position = t.positions ? load_index(t.positions, t.positions_64, i) : 0, at = -2;
    if (slot >= 0 && slot < c.sequences) {
      const int64_t length = c.lengths[slot];
      // (a sequence's end is where its last token is, while there is no room for another one)
      const bool held_back = !t.positions && (c.refused ? c.refused[slot] : *c.status) != 0;
      if (!t.positions) position = length - 1;
      at = -1;
      if (!held_back && position >= 0 && position < length && position < c.width * c.page_size) {
        const int64_t page = c.tables[slot * c.width + position / c.page_size];
        if (page >= 0 && page < c.pages) at = page * c.page_bytes + (position % c.page_size) * c.head_dim * c.item;
      }
    }
    token_at[n] = at;
    token_position[n] = position;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < here * pairs; i += kThreads) {
    const int token = i / pairs;
    table[i] = cos_sin(t.turns[i - token * pairs], token_position[token], s);
  }
  __syncthreads();
  const int unit = threadIdx.x % s.units, rest = threadIdx.x / s.units;
  const int lane = rest % s.head_lanes;
  const Unit at_unit = unit_of<W, kInterleaved>(unit, s);
  if (rest >= s.head_lanes * s.block_tokens) return;
  using Out = std::conditional_t<kE4m3, uint8_t, __nv_bfloat16>;
  const int64_t head_bytes = (int64_t)c.page_size * c.head_dim * c.item, values = c.kv_heads * head_bytes;
  for (int token = rest / s.head_lanes; token < here; token += s.block_tokens) {
    float2 cs[W];
    unit_table<W, kInterleaved>(table, token, unit, pairs, at_unit.turns, cs);
    const int64_t i = first + token, at = token_at[token];
    __nv_bfloat16* q_out = t.q_out + i * s.heads_q * s.head_dim;
    if (at == -2) {
      // (zeros whatever the row holds)
      for (int h = lane; h < s.heads_q; h += s.head_lanes) {
        if constexpr (W > 1) {
          const float zeros[W] = {};
          for (int e = unit; e < s.head_dim / W; e += s.units) Vec<__nv_bfloat16>::store(q_out + (int64_t)h * s.head_dim + e * W, zeros);
        } else {
          for (int e = unit; e < s.head_dim; e += s.units) q_out[(int64_t)h * s.head_dim + e] = __float2bfloat16_rn(0.0f);
        }
      }
      continue;
    }
    using B = __nv_bfloat16;
    constexpr bool kTwo = two_pieces<W, kInterleaved>();
    // The lane's first key and value are on their way while the queries are turned.  Values go by the keys' units, in pieces behind one another.
    const B *k = t.k + i * t.k_token, *v = t.v + i * t.v_token;
    const bool written = at >= 0 && lane < c.kv_heads;
    const int v_at = unit * W * (kTwo ? 2 : 1);
    const Unit v_unit = {min(v_at, s.head_dim - W), min(v_at + W, s.head_dim - W), false};
    Raw<B, W, kTwo> k_first, v_first;
    k_first.load(k + min(lane, c.kv_heads - 1) * t.k_head, at_unit);
    v_first.load(v + min(lane, c.kv_heads - 1) * t.v_head, v_unit);
    turn_heads<B, W, kInterleaved, 8>(t.q + i * t.q_token, t.q_head, lane, s.heads_q, s.head_lanes, at_unit, cs, [&](int h) { return PutDense<B>{q_out + (int64_t)h * s.head_dim}; });
    if (!written) continue;
    char* const row = t.layer_pool + at;
    auto put_key = [&](int h) { return PutCache<kE4m3>{reinterpret_cast<Out*>(row + h * head_bytes), kE4m3 ? t.scales[h] : 1.0f}; };
    auto put_value = [&](int h) { return PutCache<kE4m3>{reinterpret_cast<Out*>(row + values + h * head_bytes), kE4m3 ? t.scales[c.kv_heads + h] : 1.0f}; };
    turn_unit<B, W, kInterleaved>(k_first, at_unit, cs, put_key(lane));
    turn_unit<B, W, kInterleaved>(v_first, v_unit, cs, put_value(lane));
    turn_heads<B, W, kInterleaved, 8>(k, t.k_head, lane + s.head_lanes, c.kv_heads, s.head_lanes, at_unit, cs, put_key);
    turn_heads<B, W, kInterleaved, 8>(v, t.v_head, lane + s.head_lanes, c.kv_heads, s.head_lanes, v_unit, cs, put_value);
  }
}

// Threads by unit, lane of heads and token.  A thread takes four heads or more by the same cosines, unless that leaves the GPU with less than 512
// threads on each SM: then the heads are spread.
RotaryShape rotary_shape(int64_t tokens, int heads_q, int heads_k, int head_dim, int rotary_dim, bool interleaved, int wide) {
  RotaryShape s = {};
  s.heads_q = heads_q; s.heads_k = heads_k; s.head_dim = head_dim; s.rotary_dim = rotary_dim;
  s.rotary_units = wide == 1 ? rotary_dim / 2 : interleaved ? rotary_dim / wide : rotary_dim / 2 / wide;
  const int pieces = (head_dim - rotary_dim) / wide;                      // that do not turn
  s.units = s.rotary_units + (wide == 1 || !interleaved ? (pieces + 1) / 2 : pieces);
  const int rest = kThreads / s.units, heads = heads_q > heads_k ? heads_q : heads_k;
  const int64_t enough = (int64_t)device_sm_count() * 512;
  int lanes = 1;
  while (lanes * 2 <= rest && lanes < heads && (lanes * 8 <= heads || tokens * s.units * lanes < enough)) lanes *= 2;
  s.head_lanes = lanes;
  s.block_tokens = rest / lanes;
  return s;
}

// How many tokens a block takes in all: so many waves of blocks where their tables of cosines (and what else a token needs) allow it.  One for tokens that are
// all alike (1024 blocks of 8 tokens were 1.4 waves); four where some of them, the padding of a batch, may have next to nothing to do (16 prompts of 256
// to 976 tokens, bf16 48.1 us by one wave, 45.8 by four; e4m3 51.2 and 49.0.  Of 1024 tokens each, bf16 61.2 and 60.2, and e4m3, which alone has more by it, 58.3 and 64.2: which tokens
// are padding is on the device).
int32_t set_span(RotaryShape& s, int64_t tokens, const void* kernel, int token_bytes, int waves) {
  const int bytes = s.rotary_dim / 2 * (int)sizeof(float2) + token_bytes;
  const int64_t most = bytes > 0 ? 40960 / bytes : 1 << 20;
  const int64_t resident = (int64_t)device_sm_count() * resident_ctas(kernel, kThreads, 16384) * waves;
  int64_t span = ceil_div(ceil_div(tokens, resident), s.block_tokens) * s.block_tokens;
  if (span > most) span = most;
  s.span = (int32_t)span;
  return (int32_t)span * bytes;
}

bool multiple(std::initializer_list<int64_t> v, int64_t n) {
  for (const int64_t x : v) if (x % n != 0) return false;
  return true;
}

template <typename T, int W, bool kInterleaved>
cudaError_t launch_rotary(const RotaryTensors& t, RotaryShape s, cudaStream_t st) {
  const auto kernel = rotary_kernel<T, W, kInterleaved>;
  const int smem = set_span(s, t.tokens, reinterpret_cast<const void*>(kernel), 0, 1);
  return launch_overlapped(kLaunchShort, kernel, dim3((unsigned)ceil_div(t.tokens, s.span)), dim3(kThreads), (size_t)smem, st, t, s);
}

template <int W, bool kInterleaved, bool kE4m3>
cudaError_t launch_append(const AppendTensors& t, RotaryShape s, cudaStream_t st) {
  const auto kernel = append_kernel<W, kInterleaved, kE4m3>;
  const int smem = set_span(s, t.tokens, reinterpret_cast<const void*>(kernel), 16, 4);
  return launch_overlapped(kLaunchShort, kernel, dim3((unsigned)ceil_div(t.tokens, s.span)), dim3(kThreads), (size_t)smem, st, t, s);
}

}  // namespace
}  // namespace metis

using namespace metis;

extern "C" int32_t metis_rotary(const metis_rotary_args* a) {
  if (!a || !a->q || !a->q_out || !a->turns || (a->heads_k > 0 && (!a->k || !a->k_out))) return fail(METIS_ERR_BAD_ARGUMENT, "null pointer");
  if (a->dtype != METIS_DTYPE_BF16 && a->dtype != METIS_DTYPE_F32) return fail(METIS_ERR_BAD_ARGUMENT, "dtype must be bf16 or fp32");
  if (a->tokens <= 0 || a->inner <= 0 || a->heads_q <= 0 || a->heads_k < 0 || a->head_dim <= 0 || a->head_dim > 256 || a->head_dim % 8 != 0)
    return fail(METIS_ERR_BAD_SHAPE, "tokens and heads must be positive and head_dim a multiple of 8 up to 256");
  if (a->rotary_dim <= 0 || a->rotary_dim > a->head_dim || a->rotary_dim % 2 != 0)
    return fail(METIS_ERR_BAD_SHAPE, "rotary_dim must be even and at most head_dim");
  const int item = a->dtype == METIS_DTYPE_BF16 ? 2 : 4, wide = 16 / item;
  // 16 bytes at a time where the pairs, the tensors' rows and addresses allow it, element by element elsewhere
  const bool vectors = (a->interleaved ? a->rotary_dim : a->rotary_dim / 2) % wide == 0 && multiple({a->q_outer, a->q_token, a->q_head}, wide) &&
                       (a->heads_k == 0 || multiple({a->k_outer, a->k_token, a->k_head}, wide)) && aligned16(a->q) && aligned16(a->q_out) &&
                       aligned16(a->k) && aligned16(a->k_out);
  RotaryShape s = rotary_shape(a->tokens, a->heads_q, a->heads_k, a->head_dim, a->rotary_dim, a->interleaved != 0, vectors ? wide : 1);
  s.magnitude = a->magnitude;
  s.sign = a->inverse ? -1.0f : 1.0f;
  if (a->tokens >= ((int64_t)1 << 31)) return fail(METIS_ERR_TOO_LARGE, "more tokens than one launch takes");
  const RotaryTensors t = {a->positions, a->tokens, a->inner, a->turns, a->q, a->k, a->q_outer, a->q_token, a->q_head, a->k_outer, a->k_token, a->k_head,
                           a->q_out, a->k_out, a->positions_64 != 0};
  const cudaStream_t st = static_cast<cudaStream_t>(a->stream);
  const bool in = a->interleaved != 0;
  const auto by_layout = [&](auto element, auto width) {
    using T = decltype(element);
    constexpr int W = decltype(width)::value;
    return in ? launch_rotary<T, W, true>(t, s, st) : launch_rotary<T, W, false>(t, s, st);
  };
  using One = std::integral_constant<int, 1>;
  if (item == 2) METIS_CUDA_OK((vectors ? by_layout(__nv_bfloat16(), std::integral_constant<int, 8>()) : by_layout(__nv_bfloat16(), One())));
  else           METIS_CUDA_OK((vectors ? by_layout(0.0f, std::integral_constant<int, 4>()) : by_layout(0.0f, One())));
  count_rollout_launches(1);
  return METIS_OK;
}

extern "C" int32_t metis_cache_append(const metis_cache* cache, const metis_append_args* a) {
  AppendTensors t = {};
  if (const int32_t rc = check_cache(cache, &t.cache)) return rc;
  const CacheView& c = t.cache;
  if (!a || !a->k || !a->v || (a->heads_q > 0 && (!a->q || !a->q_out))) return fail(METIS_ERR_BAD_ARGUMENT, "null pointer");
  if (a->tokens <= 0 || a->heads_q < 0 || a->layer < 0 || a->layer >= c.layers) return fail(METIS_ERR_BAD_SHAPE, "tokens must be positive and the layer one of the cache");
  if (a->turns && (a->rotary_dim <= 0 || a->rotary_dim > c.head_dim || a->rotary_dim % 2 != 0)) return fail(METIS_ERR_BAD_SHAPE, "rotary_dim must be even and at most head_dim");
  if (!multiple({a->k_token, a->k_head, a->v_token, a->v_head}, 8) || (a->heads_q > 0 && !multiple({a->q_token, a->q_head}, 8)))
    return fail(METIS_ERR_BAD_ALIGNMENT, "strides must be multiples of 8 elements");
  if (!aligned16(a->k) || !aligned16(a->v) || !aligned16(a->q) || !aligned16(a->q_out)) return fail(METIS_ERR_BAD_ALIGNMENT, "tensors must be 16-byte aligned");
  const int rotary = a->turns ? a->rotary_dim : 0;
  const bool in = a->interleaved != 0 && rotary > 0, vectors = (in ? rotary : rotary / 2) % 8 == 0;
  RotaryShape s = rotary_shape(a->tokens, a->heads_q, c.kv_heads, c.head_dim, rotary, in, vectors ? 8 : 1);
  s.heads_q = a->heads_q;
  s.magnitude = a->magnitude;
  s.sign = 1.0f;
  if (a->tokens >= ((int64_t)1 << 31)) return fail(METIS_ERR_TOO_LARGE, "more tokens than one launch takes");
  const int64_t part = (int64_t)c.kv_heads * c.page_size * c.head_dim * c.item;       // keys, or values, of one layer on a page
  t.layer_pool = c.pool + a->layer * 2 * part;
  t.scales = cache->scales ? cache->scales + (int64_t)a->layer * 2 * c.kv_heads : nullptr;
  t.slots = a->slots; t.positions = a->positions; t.tokens = a->tokens; t.turns = a->turns;
  t.q = static_cast<const __nv_bfloat16*>(a->q); t.k = static_cast<const __nv_bfloat16*>(a->k); t.v = static_cast<const __nv_bfloat16*>(a->v);
  t.q_token = a->q_token; t.q_head = a->q_head; t.k_token = a->k_token; t.k_head = a->k_head; t.v_token = a->v_token; t.v_head = a->v_head;
  t.q_out = static_cast<__nv_bfloat16*>(a->q_out);
  t.slots_64 = (a->index_64 & 1) != 0; t.positions_64 = (a->index_64 & 2) != 0;
  const cudaStream_t st = static_cast<cudaStream_t>(a->stream);
  const bool e4m3 = c.item == 1;
  const auto by_layout = [&](auto width) {
    constexpr int W = decltype(width)::value;
    return in ? (e4m3 ? launch_append<W, true, true>(t, s, st) : launch_append<W, true, false>(t, s, st))
              : (e4m3 ? launch_append<W, false, true>(t, s, st) : launch_append<W, false, false>(t, s, st));
  };
  METIS_CUDA_OK((vectors ? by_layout(std::integral_constant<int, 8>()) : by_layout(std::integral_constant<int, 1>())));
  count_rollout_launches(1);
  return METIS_OK;
}
