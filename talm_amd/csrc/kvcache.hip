// A layer's 8-bit key and value cache for gfx950: new tokens are written into it, read back, and
// attended to.
//
// A sequence's tokens form blocks of 64. A complete block is a page of the pool: its keys and its
// values, per KV head, as e4m3 codes times one power of two, the smallest that takes the block's
// largest magnitude to at most 448 (a floating code: columns of the keys that are many times louder
// than the others cost those no precision; a power of two: x / scale is exact, so a code does not
// depend on how the division is done). The tokens behind the last complete block stay in 16 bits
// (the tail), so what a cache holds does not depend on how its tokens were split over calls, and no
// code is ever scaled again.
//
// A page lies in the order in which the attention's matrix instructions take it, a lane's 16 bytes
// behind each other and a wavefront's 1 KiB too:
//   keys    [tile of 16 tokens 4][64 columns D/64][quarter of them 4][token 16][column 16]
//   values  [tile of 16 columns D/16][g 4][column 16][tile of tokens 4][r 4], token = 16 tile + 4 g + r
// S^T = K Q^T leaves lane (g, column) with tokens 16 tile + 4 g + r of its query; the values' order
// makes the same tokens the lane's share of P^T in O^T = V^T P^T, so P never leaves its registers.
#include <math.h>

#include <algorithm>
#include <type_traits>

#include "common.h"

namespace talm {
namespace {

typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef _Float16 half4 __attribute__((ext_vector_type(4)));
typedef _Float16 half2_ __attribute__((ext_vector_type(2)));
typedef __bf16 bf8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf2 __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

constexpr int kBlock = 64;     // tokens of a page
constexpr int kThreads = 256;
constexpr int kWaves = kThreads / kWave;
// the most workgroups of a launch's axis: its threads are counted in 32 bits
constexpr int64_t kGrid = 0xffffffffll / kThreads;
constexpr int kSplits = 256;   // the most parts that the keys of a row are split into
constexpr int kNear = 4;       // tiles beside each other that share a die's L2

struct Cache {
  const uint8_t* codes;   // [pages, 2, kv, 64 D]
  const float* scales;    // [pages, 2, kv]
  const uint16_t* tail;   // [n_seqs, 2, kv, 64 D]: keys [64, D], values [D, 64]
  const int32_t* table;   // [n_seqs, width]
  int64_t n_pages;
  int width, n_seqs, kv;
  __device__ __forceinline__ int64_t page(int seq, int block) const {
    // -1 for what is no page of the pool
    const int64_t p = block < width ? table[static_cast<int64_t>(seq) * width + block] : -1;
    return p < n_pages ? p : -1;
  }
};

// A sequence's new rows [row0, row0 + n) behind `past` tokens, kept inside the buffers' rows, the
// caller's longest counts and the table whatever the device arrays hold.
struct Span {
  int row0, past, n;
};
__device__ __forceinline__ Span span_of(int lo, int hi, int past, int n_rows, int max_new, int max_len) {
  lo = max(0, min(lo, n_rows));
  hi = max(lo, min(hi, n_rows));
  if (past < 0 || past >= max_len) return Span{lo, 0, 0};
  return Span{lo, past, min(min(hi - lo, max_new), max_len - past)};
}
__device__ __forceinline__ Span span_of(const int32_t* bounds, const int32_t* past, int seq, int64_t n_rows,
                                        int max_new, int max_len) {
  return span_of(bounds[2 * seq], bounds[2 * seq + 1], past[seq], static_cast<int>(n_rows), max_new, max_len);
}

// kMost: the type's largest number. Attention holds sums of values times kUnit: bfloat16's largest values times
// weights below 2^8 of at most 2^30 tokens would leave fp32 (2^-40 costs results below 2^-100 bits).
struct F16 {
  static constexpr float kMost = 65504.f, kUnit = 1.f;
  static __device__ __forceinline__ float up(uint32_t bits) { return h2f(static_cast<uint16_t>(bits)); }
  static __device__ __forceinline__ uint16_t down(float x) { return f2h(x); }
  // 8 e4m3 codes, exactly
  static __device__ __forceinline__ half8 codes(u32x2 w) {
    const half2_ a = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w.x, 1.f, false);
    const half2_ b = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w.x, 1.f, true);
    const half2_ c = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w.y, 1.f, false);
    const half2_ d = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w.y, 1.f, true);
    return half8{a.x, a.y, b.x, b.y, c.x, c.y, d.x, d.y};
  }
  static __device__ __forceinline__ f32x4 mfma(half8 a, half8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
  }
  static __device__ __forceinline__ f32x16 mfma(half8 a, half8 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
  }
};
struct BF16 {
  static constexpr float kMost = 0x1.fep127f, kUnit = 0x1p-40f;
  static __device__ __forceinline__ float up(uint32_t bits) { return __builtin_bit_cast(float, bits << 16); }
  static __device__ __forceinline__ uint16_t down(float x) {
    return __builtin_bit_cast(uint16_t, static_cast<__bf16>(x));
  }
  static __device__ __forceinline__ half8 codes(u32x2 w) {
    const bf2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w.x, 1.f, false);
    const bf2 b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w.x, 1.f, true);
    const bf2 c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w.y, 1.f, false);
    const bf2 d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w.y, 1.f, true);
    return __builtin_bit_cast(half8, bf8{a.x, a.y, b.x, b.y, c.x, c.y, d.x, d.y});
  }
  static __device__ __forceinline__ f32x4 mfma(half8 a, half8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf8, a), __builtin_bit_cast(bf8, b), c, 0, 0,
                                                   0);
  }
  static __device__ __forceinline__ f32x16 mfma(half8 a, half8 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf8, a), __builtin_bit_cast(bf8, b), c, 0, 0,
                                                   0);
  }
};

// ------------------------------------------------------------------------------------------------
// Writing
// ------------------------------------------------------------------------------------------------

struct WriteArgs {
  const uint16_t* k;
  int64_t k_tok, k_head;
  const uint16_t* v;
  int64_t v_tok, v_head;
  int64_t n_rows;
  const int32_t* bounds;
  const int32_t* past;
  int max_new, max_len, chunks;  // chunks: blocks that a sequence's new tokens can touch
  uint8_t* codes;
  float* scales;
  uint16_t* tail;
  Cache c;  // the same buffers
  const float* cos;  // with rotary positions, rows of cs_tok
  const float* sin;
  int64_t cs_tok;
  const uint16_t* q;
  int64_t q_tok, q_head;
  int n_q;
  uint16_t* q_out;  // [n_rows, n_q, D]
  int64_t kv_items;  // workgroups of the cache; those behind them turn the queries
  uint32_t first;    // the launch's first workgroup of all
};

// Columns [d, d + 8) of a row of D, turned (the pair of column d is d + D/2 or d - D/2).
template <class T, int D>
__device__ __forceinline__ void row8(const uint16_t* row, const float* cos, const float* sin, int d, bool turn,
                                     uint32_t (&out)[4]) {
  const u32x4 w = *reinterpret_cast<const u32x4*>(row + d);
  if (!turn) {
#pragma unroll
    for (int i = 0; i < 4; ++i) out[i] = w[i];
    return;
  }
  const bool first = d < D / 2;
  const u32x4 p = *reinterpret_cast<const u32x4*>(row + (first ? d + D / 2 : d - D / 2));
  float cs[8], sn[8];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const f32x4 a = reinterpret_cast<const f32x4*>(cos + d)[i], b = reinterpret_cast<const f32x4*>(sin + d)[i];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      cs[4 * i + j] = a[j];
      sn[4 * i + j] = b[j];
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    uint32_t bits = 0;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const float x = T::up((w[i] >> (16 * j)) & 0xffffu), y = T::up((p[i] >> (16 * j)) & 0xffffu);
      const float c = cs[2 * i + j], s = sn[2 * i + j];
      const float z = first ? x * c - y * s : x * c + y * s;
      bits |= static_cast<uint32_t>(T::down(z)) << (16 * j);
    }
    out[i] = bits;
  }
}

// A block's scale from its largest finite magnitude: 2^e, e the smallest with top <= 448 2^e (448 =
// 1.75 * 2^8); 1 for a block of zeros. e is at least -100, which only magnitudes below 2^-91 meet.
__device__ __forceinline__ float block_scale(float top) {
  const uint32_t bits = __builtin_bit_cast(uint32_t, top);
  int e = static_cast<int>(bits >> 23) - 127 - 8;
  if ((bits & 0x7fffffu) > 0x600000u) ++e;
  e = max(e, -100);
  return top > 0.f ? __builtin_bit_cast(float, static_cast<uint32_t>(e + 127) << 23) : 1.f;
}

// 1 / scale of a power of two
__device__ __forceinline__ float inverse(float scale) {
  return __builtin_bit_cast(float, (254u << 23) - __builtin_bit_cast(uint32_t, scale));
}

__device__ __forceinline__ float finite_or_nan(float x) {
  return fabsf(x) < __builtin_inff() ? x : __builtin_nanf("");
}

template <class T>
__device__ __forceinline__ uint32_t code4(uint32_t lo, uint32_t hi, float inv) {
  float x[4] = {T::up(lo & 0xffffu), T::up(lo >> 16), T::up(hi & 0xffffu), T::up(hi >> 16)};
#pragma unroll
  for (int i = 0; i < 4; ++i) x[i] = finite_or_nan(x[i]) * inv;
  int w = __builtin_amdgcn_cvt_pk_fp8_f32(x[0], x[1], 0, false);
  w = __builtin_amdgcn_cvt_pk_fp8_f32(x[2], x[3], w, true);
  return static_cast<uint32_t>(w);
}

template <class T>
__device__ __forceinline__ float top_of(const uint32_t (&w)[4], float top) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float a = fabsf(T::up(w[i] & 0xffffu)), b = fabsf(T::up(w[i] >> 16));
    if (a < __builtin_inff()) top = fmaxf(top, a);
    if (b < __builtin_inff()) top = fmaxf(top, b);
  }
  return top;
}

// One workgroup: block `j` behind past's of one sequence, one KV head, keys or values. A complete
// block becomes a page; the workgroup of the first block, the one that reads the tail, then also
// stores the tokens behind the last complete block into it, so no other touches the tail. A block has one
// scale, so its workgroup holds it whole (LDS, where the page's order is made too) and reads it once.
//
// Bound by its bytes where it is large: 32001 tokens in bfloat16 with 12 query heads turned, 279 MB, take 58 us
// (4.8 TB/s; a large copy reaches 5.2), four prompts of 1531 to 4096 tokens in fp16, 111 MB, 22; by the launch
// and a chain of cache misses (arguments, the sequence's numbers, rows) where it is small: one token 2.9 us, one
// of each of 64 sequences 6.2, of which those that complete a block first read its 63 others from the tail.
template <class T, int D, bool kTurn>
__global__ __launch_bounds__(kThreads) void cache_write_kernel(WriteArgs a) {
  constexpr int kPer = D / 8;  // 16-byte pieces of a row
  __shared__ alignas(16) uint16_t tile[kBlock][D + 2];
  __shared__ float tops[kWaves];
  const int tid = threadIdx.x, lane = tid & 63;
  const uint32_t item = a.first + blockIdx.x;
  if (kTurn && item >= a.kv_items) {
    const int64_t i = (item - a.kv_items) * kThreads + tid;
    if (i >= a.n_rows * a.n_q * kPer) return;
    const int d = static_cast<int>(i % kPer) * 8;
    const int64_t rh = i / kPer, row = rh / a.n_q;
    const int head = static_cast<int>(rh - row * a.n_q);
    uint32_t w[4];
    row8<T, D>(a.q + row * a.q_tok + head * a.q_head, a.cos + row * a.cs_tok, a.sin + row * a.cs_tok, d, true, w);
    *reinterpret_cast<u32x4*>(a.q_out + rh * D + d) = u32x4{w[0], w[1], w[2], w[3]};
    return;
  }
  const int rest = static_cast<int>(item / static_cast<unsigned>(a.chunks));
  const int j = static_cast<int>(item) - rest * a.chunks;
  const int seq = (rest >> 1) / a.c.kv, head = (rest >> 1) - seq * a.c.kv, which = rest & 1;
  // the arguments in one cache miss, the sequence's numbers in the next
  asm volatile("" ::"s"(a.bounds), "s"(a.past), "s"(a.n_rows), "s"(a.max_new), "s"(a.max_len), "s"(a.tail),
               "s"(a.k), "s"(a.k_tok), "s"(a.k_head), "s"(a.v), "s"(a.v_tok), "s"(a.v_head));
  const int lo_row = a.bounds[2 * seq], hi_row = a.bounds[2 * seq + 1], held = a.past[seq];
  asm volatile("" ::"s"(lo_row), "s"(hi_row), "s"(held));
  const Span s = span_of(lo_row, hi_row, held, static_cast<int>(a.n_rows), a.max_new, a.max_len);
  const int len = s.past + s.n;
  const int block = s.past / kBlock + j, last = len / kBlock;  // last: the open block, perhaps empty
  if (s.n == 0 || (j > 0 && block >= last)) return;
  const int64_t slot = (static_cast<int64_t>(seq) * 2 + which) * a.c.kv + head;
  uint16_t* tail = a.tail + slot * (kBlock * D);
  const uint16_t* src = (which ? a.v : a.k) + head * (which ? a.v_head : a.k_head);
  const int64_t tok = which ? a.v_tok : a.k_tok;
  const bool turn = kTurn && which == 0;
  // the 8 columns from d on of the sequence's token `t`, a new one
  auto fresh = [&](int t, int d, uint32_t (&w)[4]) {
    const int64_t row = s.row0 + (t - s.past);  // of the operands
    row8<T, D>(src + row * tok, kTurn ? a.cos + row * a.cs_tok : nullptr, kTurn ? a.sin + row * a.cs_tok : nullptr,
               d, turn, w);
  };
  if (block < last) {
    const int64_t page = a.c.page(seq, block);
    // the block to LDS: what the tail has of it in 16-byte pieces (8 columns of a key, 8 tokens of a
    // column of the values), then the new tokens in pieces of 8 columns
    float top = 0.f;
    const int old = max(s.past - block * kBlock, 0);
    u32x4 x[kBlock * kPer / kThreads];
    if (old > 0) {
#pragma unroll
      for (int n = 0; n < kBlock * kPer / kThreads; ++n)
        x[n] = reinterpret_cast<const u32x4*>(tail)[n * kThreads + tid];
    }
    for (int i = old * kPer + tid; i < kBlock * kPer; i += kThreads) {
      const int t = i / kPer, d = (i % kPer) * 8;
      uint32_t w[4];
      fresh(block * kBlock + t, d, w);
      top = top_of<T>(w, top);
#pragma unroll
      for (int e = 0; e < 4; ++e) *reinterpret_cast<uint32_t*>(&tile[t][d + 2 * e]) = w[e];
    }
    if (old > 0) {
#pragma unroll
      for (int n = 0; n < kBlock * kPer / kThreads; ++n) {
        const int i = n * kThreads + tid;
        if (which == 0) {
          const int t = i / kPer, d = (i % kPer) * 8;
          uint32_t w[4] = {x[n].x, x[n].y, x[n].z, x[n].w};
          if (t < old) {
            top = top_of<T>(w, top);
#pragma unroll
            for (int e = 0; e < 4; ++e) *reinterpret_cast<uint32_t*>(&tile[t][d + 2 * e]) = w[e];
          }
        } else {
          const int d = i / (kBlock / 8), t = (i % (kBlock / 8)) * 8;
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const uint16_t y = static_cast<uint16_t>(x[n][e / 2] >> (16 * (e % 2)));
            if (t + e < old) {
              const float z = fabsf(T::up(y));
              if (z < __builtin_inff()) top = fmaxf(top, z);
              tile[t + e][d] = y;
            }
          }
        }
      }
    }
    top = wave_max(top);
    if (lane == 0) tops[tid / kWave] = top;
    __syncthreads();
    top = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]));
    const float scale = block_scale(top), inv = inverse(scale);
    if (page >= 0) {
      const int64_t place = (page * 2 + which) * a.c.kv + head;
      if (tid == 0) a.scales[place] = scale;
      u32x4* dst = reinterpret_cast<u32x4*>(a.codes + place * (kBlock * D));
      for (int i = tid; i < kBlock * D / 16; i += kThreads) {
        const int row = i & 15, g = (i >> 4) & 3, outer = i >> 6;
        u32x4 w;
        if (which == 0) {
          constexpr int kC = D / 64;
          const int t = (outer / kC) * 16 + row, d = (outer % kC) * 64 + g * 16;
          const uint32_t* x = reinterpret_cast<const uint32_t*>(&tile[t][d]);
#pragma unroll
          for (int e = 0; e < 4; ++e) w[e] = code4<T>(x[2 * e], x[2 * e + 1], inv);
        } else {
          const int d = outer * 16 + row;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int t = e * 16 + g * 4;
            w[e] = code4<T>(tile[t][d] | static_cast<uint32_t>(tile[t + 1][d]) << 16,
                            tile[t + 2][d] | static_cast<uint32_t>(tile[t + 3][d]) << 16, inv);
          }
        }
        dst[i] = w;
      }
    }
  }
  if (j > 0) return;
  // the open block's new tokens; what the first block took from the tail was read before its barrier
  const int lo = max(last * kBlock, s.past);
  for (int i = tid; i < (len - lo) * kPer; i += kThreads) {
    const int at = lo + i / kPer, d = (i % kPer) * 8, t = at - last * kBlock;
    uint32_t w[4];
    fresh(at, d, w);
    if (which == 0) {
      *reinterpret_cast<u32x4*>(tail + t * D + d) = u32x4{w[0], w[1], w[2], w[3]};
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        tail[(d + 2 * e) * kBlock + t] = static_cast<uint16_t>(w[e] & 0xffffu);
        tail[(d + 2 * e + 1) * kBlock + t] = static_cast<uint16_t>(w[e] >> 16);
      }
    }
  }
}

// ------------------------------------------------------------------------------------------------
// Reading back
// ------------------------------------------------------------------------------------------------

struct ReadArgs {
  Cache c;
  const int32_t* length;
  const int32_t* bounds;
  const int32_t* past;
  int64_t n_rows;
  int max_new, max_len, chunks;
  uint16_t* k;  // [n_rows, kv, D]
  uint16_t* v;
  uint32_t first;  // the launch's first workgroup of all
};

// A lane's 16 codes times their scale in 16 bits. A value near the type's largest number may have been rounded
// up to a power of two that the type does not hold (with the largest scale only): its largest number
// stands for it.
template <class T>
__device__ __forceinline__ void held(u32x4 w, float scale, uint32_t (&out)[8]) {
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    if constexpr (__is_same(T, F16)) {
      out[2 * e] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w[e], scale, false));
      out[2 * e + 1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w[e], scale, true));
    } else {
      out[2 * e] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w[e], scale, false));
      out[2 * e + 1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w[e], scale, true));
    }
  }
  constexpr uint32_t kInf = __is_same(T, F16) ? 0x7c00u : 0x7f80u;
  if (scale >= (__is_same(T, F16) ? 0x1p8f : 0x1p120f)) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      if ((out[e] & 0x7fffu) == kInf) out[e] -= 1;
      if ((out[e] & 0x7fff0000u) == kInf << 16) out[e] -= 0x10000u;
    }
  }
}

// One workgroup: one block of one sequence, one KV head, keys or values. A lane's 16 keys are one token's
// columns and go where they belong; its values are 16 tokens of one column and are turned in LDS. Bound by its
// bytes: 16 sequences of 4000 to 8191 tokens in bfloat16, 153 MB, take 32 us (4.8 TB/s of a copy's 5.2); 8
// of 100 to 500 with heads of 64, 2 MB, take 4.9.
template <class T, int D>
__global__ __launch_bounds__(kThreads) void cache_read_kernel(ReadArgs a) {
  constexpr int kPer = D / 8, kEach = kBlock * D / 16 / kThreads;
  __shared__ alignas(16) uint16_t tile[kBlock][D + 8];
  const int tid = threadIdx.x;
  const uint32_t item = a.first + blockIdx.x;
  const int j = static_cast<int>(item % a.chunks);
  const int rest = static_cast<int>(item / a.chunks);
  const int which = rest & 1, head = (rest >> 1) % a.c.kv, seq = (rest >> 1) / a.c.kv;
  const Span s = span_of(a.bounds, a.past, seq, a.n_rows, a.max_new, a.max_len);
  const int len = min(max(a.length[seq], 0), a.max_len);
  const int block = s.past / kBlock + j, first = block * kBlock;
  const int lo = max(first, s.past), hi = min(first + kBlock, s.past + s.n);
  if (lo >= hi) return;
  const int64_t pitch = static_cast<int64_t>(a.c.kv) * D;
  // token t's row
  uint16_t* dst = (which ? a.v : a.k) + static_cast<int64_t>(s.row0 - s.past) * pitch + head * D;
  const int64_t page = block < len / kBlock ? a.c.page(seq, block) : -1;
  if (page >= 0) {
    const int64_t place = (page * 2 + which) * a.c.kv + head;
    const float scale = a.c.scales[place];
    const u32x4* src = reinterpret_cast<const u32x4*>(a.c.codes + place * (kBlock * D));
    u32x4 w[kEach];
#pragma unroll
    for (int n = 0; n < kEach; ++n) w[n] = __builtin_nontemporal_load(src + n * kThreads + tid);
#pragma unroll
    for (int n = 0; n < kEach; ++n) {
      const int i = n * kThreads + tid, row = i & 15, g = (i >> 4) & 3, outer = i >> 6;
      uint32_t x[8];
      held<T>(w[n], scale, x);
      if (which == 0) {
        constexpr int kC = D / 64;
        const int at = first + (outer / kC) * 16 + row, d = (outer % kC) * 64 + g * 16;
        if (at >= lo && at < hi) {
          u32x4* to = reinterpret_cast<u32x4*>(dst + at * pitch + d);
          to[0] = u32x4{x[0], x[1], x[2], x[3]};
          to[1] = u32x4{x[4], x[5], x[6], x[7]};
        }
      } else {
        const int d = outer * 16 + row;
#pragma unroll
        for (int e = 0; e < 16; ++e)
          tile[e / 4 * 16 + g * 4 + e % 4][d] = static_cast<uint16_t>(x[e / 2] >> (16 * (e % 2)));
      }
    }
    if (which == 0) return;
  } else {
    // the open block's tokens from the tail (the keys in the order of the tile, the values transposed),
    // zeros behind them and where there is no page
    const bool open = block == len / kBlock;
    const uint16_t* tail = a.c.tail + ((static_cast<int64_t>(seq) * 2 + which) * a.c.kv + head) * (kBlock * D);
    for (int i = tid; i < kBlock * D; i += kThreads) {
      const int t = which ? i % kBlock : i / D, d = which ? i / kBlock : i % D;
      tile[t][d] = open && first + t < len ? tail[i] : 0;
    }
  }
  __syncthreads();
  for (int i = tid; i < (hi - lo) * kPer; i += kThreads) {
    const int at = lo + i / kPer, d = (i % kPer) * 8;
    *reinterpret_cast<u32x4*>(dst + at * pitch + d) = *reinterpret_cast<const u32x4*>(&tile[at - first][d]);
  }
}

// ------------------------------------------------------------------------------------------------
// Attention
// ------------------------------------------------------------------------------------------------

struct AttnArgs {
  Cache c;
  const int32_t* bounds;
  const int32_t* past;
  int n_rows, max_new, max_len;
  int n_q, group, group_magic, group_shift;  // query heads per KV head; row / group is over() of them
  int cols, splits, per;  // rows of a tile; parts of the pages, pages of a part
  int turn;               // 2^n - 1 below both 8 and `splits`
  bool listed;            // the grid's first axis: the sequences' tiles in a row, else one tile each
  int window, sinks;  // window 0: every key
  float scale_log2;
  const uint16_t* q;
  int64_t q_tok, q_head;
  uint16_t* out;      // [n_rows, n_q, D]
  float* part_o;      // [n_rows, n_q, splits, D]
  float2* part_ml;    // [n_rows, n_q, splits]: maximum, sum
  // n / group of 0 <= n < 2^30: the integer division would be some thirty instructions in front of the
  // first load
  __device__ __forceinline__ int over(int n) const {
    return group == 1 ? n
                      : static_cast<int>(__umulhi(static_cast<uint32_t>(n), static_cast<uint32_t>(group_magic)) >>
                                         group_shift);
  }
};

// The pages that rows at places [lo, hi] see, as a list: the sinks', then the window's.
struct Visits {
  int sinks, first, count;
  __device__ __forceinline__ Visits(int lo, int hi, int window, int n_sinks) {
    const int pages = hi / kBlock + 1;
    first = window > 0 ? max(lo - window + 1, 0) / kBlock : 0;
    sinks = window > 0 ? min((n_sinks + kBlock - 1) / kBlock, first) : 0;
    count = sinks + pages - first;
  }
  __device__ __forceinline__ int page(int i) const { return i < sinks ? i : i - sinks + first; }
};

// Four outputs in 16 bits from means of values times kUnit. A mean past the type's largest number (values whose
// codes were rounded past it) is that number, as those values are where they are read back.
template <class T>
__device__ __forceinline__ u32x2 outputs(f32x4 x) {
  constexpr float kTop = T::kMost * T::kUnit;
  if (fmaxf(fmaxf(fabsf(x[0]), fabsf(x[1])), fmaxf(fabsf(x[2]), fabsf(x[3]))) > kTop) {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (fabsf(x[e]) < __builtin_inff()) x[e] = fminf(fmaxf(x[e], -kTop), kTop);
  }
  uint32_t w[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) w[e] = T::down(x[e] * (1.f / T::kUnit));
  return u32x2{w[0] | w[1] << 16, w[2] | w[3] << 16};
}

// How S^T = K Q^T and O^T = V^T P^T of one page lie in a wavefront with kCol query columns, 16
// (v_mfma_*_16x16x32) or 32 (v_mfma_*_32x32x16; half as many instructions for the same products, each of
// which takes the VALU's issue for about 8 cycles). Lane l is column l % kCol, quarter or half g = l / kCol.
// Its scores in order, i = 0, 1, ..: token kStep (i / 4) + 4 g + i % 4; its output columns likewise.
template <int D, int kCol>
struct Lay {
  static constexpr int kStep = kCol == 16 ? 16 : 8;
  static constexpr int kLane = kBlock * kCol / kWave;  // scores of a lane
  static constexpr int kTiles = kBlock / kCol;         // tiles of scores
  static constexpr int kEach = kLane / kTiles;         // and numbers of one
  static constexpr int kOuts = D / kCol;               // tiles of outputs, kEach numbers each
  static constexpr int kFrags = D * kCol / 512;        // operands of 8 of a row's columns
  static constexpr int kPs = kLane / 8;                // operands of P
  using Tile = typename std::conditional<kCol == 16, f32x4, f32x16>::type;
  // first column of a lane's f-th operand of a query or key row
  static __device__ __forceinline__ int column(int f, int g) {
    return kCol == 16 ? f / 2 * 64 + g * 16 + f % 2 * 8 : f / 4 * 64 + f / 2 % 2 * 32 + g * 16 + f % 2 * 8;
  }
  // places of a lane's 16 bytes in a page, without the lane's own part: the i-th load of the keys belongs
  // to tile i / (kFrags / 2) and to operands 2 (i % (kFrags / 2)) and one behind it
  static __device__ __forceinline__ int key_at(int i) {
    if (kCol == 16) return i * 64;
    constexpr int kC = D / 64;
    const int tile = i / (2 * kC), rest = i % (2 * kC);
    return (2 * tile * kC + rest / 2) * 64 + rest % 2 * 32;
  }
  static __device__ __forceinline__ int key_lane(int lane) {
    return kCol == 16 ? lane : (lane >> 4 & 1) * (D / 64) * 64 + (lane >> 5) * 16 + (lane & 15);
  }
  static __device__ __forceinline__ int value_at(int i) { return kCol == 16 ? i * 64 : i / 2 * 128 + i % 2 * 32; }
  static __device__ __forceinline__ int value_lane(int lane) {
    return kCol == 16 ? lane : (lane >> 4 & 1) * 64 + (lane >> 5) * 16 + (lane & 15);
  }
  // the codes of output tile n that meet the u-th operand of P
  static __device__ __forceinline__ u32x2 value_codes(const u32x4 (&w)[D / 16], int n, int u) {
    if constexpr (kCol == 16) return u32x2{w[n][2 * u], w[n][2 * u + 1]};
    else return u32x2{w[2 * n][u], w[2 * n + 1][u]};
  }
  // over the lanes of one column
  static __device__ __forceinline__ float max_of(float x) {
    if (kCol == 16) {
      const uint32_t u = __builtin_bit_cast(uint32_t, x);
      const auto r = __builtin_amdgcn_permlane16_swap(u, u, false, false);
      x = fmaxf(__builtin_bit_cast(float, static_cast<uint32_t>(r[0])),
                __builtin_bit_cast(float, static_cast<uint32_t>(r[1])));
    }
    const uint32_t w = __builtin_bit_cast(uint32_t, x);
    const auto q = __builtin_amdgcn_permlane32_swap(w, w, false, false);
    return fmaxf(__builtin_bit_cast(float, static_cast<uint32_t>(q[0])),
                 __builtin_bit_cast(float, static_cast<uint32_t>(q[1])));
  }
  static __device__ __forceinline__ float sum_of(float x) {
    if (kCol == 16) x += __shfl_xor(x, 16, kWave);
    return x + __shfl_xor(x, 32, kWave);
  }
};

// A workgroup: kCols = kCol kWide (token, head) rows of one sequence and KV head, the columns of S^T =
// K Q^T, against one part of its pages. Each of kWide groups of wavefronts has kCol of the columns; the
// wavefronts of a group take a page each at a time, with a running reference and sums of their own, joined
// through LDS.
//
// Weights are exp2(c s - ref) of a reference that follows the running maximum only where a score passes it
// by more than 2^8: they stay below 2^8, far inside fp16, and nearly every page leaves the sums so far as
// they are.
//
// Tiles of 16 rows, for sequences of a token or two: the pages come from memory once, and that is the time. One
// token of each of 64 sequences of 201 to 8191 tokens, 143 MB, takes 30 us (4.8 TB/s of a copy's 5.2) and 4 for
// the join; one over 131001, 67 MB, 14.5 and 4; one over 4001 5.8 and 3.3, where the start is most of it.
// Tiles of 32 and 64 rows: issue is the largest share of the time. A wavefront's page of 32 rows takes some 485
// issue slots of 4 cycles (bfloat16 535): 128 conversions of codes, 150 for the softmax (an exponential has two),
// 64 of the 32 MFMAs, the loads, and its share of the start and the join. 512 rows of 6 heads each over 8289
// tokens 40 us (630 TF/s) and 6 for the join: 25 of issue at the clock of this load, 4.4 until all workgroups
// run, and ends that spread over 14. The next turns of 12 conversations (1 to 300 tokens behind 300 to 3500) 56 us
// (580 TF/s), 35 of them issue. Converted pages shared through LDS, and 64 columns a wavefront on one wavefront
// a SIMD, were no faster (the same; 62 against 48 us with the join).
template <class T, int D, int kCol, int kWide>
__global__ __launch_bounds__(kThreads, kCol == 16 ? 3 : 2) void cache_attn_kernel(AttnArgs a) {
  using L = Lay<D, kCol>;
  using Tile = typename L::Tile;
  constexpr int kPitch = D + 4, kCols = kCol * kWide, kDeep = kWaves / kWide, kLoads = D / 16;
  constexpr bool kUnits = __is_same(T, F16);
  __shared__ float part[kDeep][kCols][kPitch];
  __shared__ float stat[2][kDeep][kCols];
  const int tid = threadIdx.x, lane = tid & 63, col = lane % kCol, g = lane / kCol;
  const int wave = __builtin_amdgcn_readfirstlane(tid / kWave), wide = wave % kWide, deep = wave / kWide;
  const int head = blockIdx.y;
  int tile = 0, seq = blockIdx.z, split = blockIdx.x;
  if (a.listed) {
    // Workgroups go to the eight dies in turn. kNear tiles beside each other, of the same part, go to one, whose
    // L2 then has their pages (20 tokens of each of 40 sequences of 2000: 41 us spread out, 30 so)
    const int slot = split >> 3;
    if (split < static_cast<int>(gridDim.x & ~(8u * kNear - 1)))
      split = (slot & ~(kNear - 1)) * 8 + (split & 7) * kNear + (slot & (kNear - 1));
    tile = split & (kNear - 1);
    split /= kNear;
    const int q = split / a.splits;
    tile += q * kNear;
    split -= q * a.splits;
  }
  // other sequences' parts in turn: a die would have the same part of every one, and later parts are those that
  // short sequences lack
  if (!a.listed) {
    split += (head + seq) & a.turn;
    if (split >= a.splits) split -= a.splits;
  }
  // A workgroup begins with a chain of cache misses; all arguments in one, the sequence's numbers and its
  // pages' places (without a window known from the part alone) in the next, then the pages.
  asm volatile("" ::"s"(a.c.codes), "s"(a.c.scales), "s"(a.c.tail), "s"(a.c.table), "s"(a.c.width), "s"(a.c.kv),
               "s"(a.bounds), "s"(a.past), "s"(a.n_rows), "s"(a.max_new), "s"(a.max_len), "s"(a.group),
               "s"(a.group_magic), "s"(a.group_shift), "s"(a.window), "s"(a.sinks), "s"(a.q), "s"(a.q_tok),
               "s"(a.q_head));
  const bool alone = kCol == 16 || a.c.n_seqs == 1;  // the sequence is known from the grid
  int early = -1;
  if (alone && a.window == 0) {
    const int mine = split * a.per + deep + kDeep * lane;
    if (mine < a.c.width) early = a.c.table[static_cast<int64_t>(seq) * a.c.width + mine];
  }
  Span s;
  if (alone) {
    const int lo_row = a.bounds[2 * seq], hi_row = a.bounds[2 * seq + 1], held = a.past[seq];
    asm volatile("" ::"s"(lo_row), "s"(hi_row), "s"(held));
    s = span_of(lo_row, hi_row, held, a.n_rows, a.max_new, a.max_len);
  } else {
    // Tile `tile` of the sequences' tiles in a row, of every 64 sequences those with the most pages first: a
    // long one that began last would be the call's tail. Lane l has sequence l's tiles.
    for (seq = 0;; seq += kWave) {
      if (seq >= a.c.n_seqs) return;
      Span mine{0, 0, 0};
      if (seq + lane < a.c.n_seqs) mine = span_of(a.bounds, a.past, seq + lane, a.n_rows, a.max_new, a.max_len);
      const int count = (mine.n * a.group + kCols - 1) / kCols;
      const int order = (mine.past + mine.n) / kBlock * kWave + kWave - 1 - lane;  // no two alike
      int before = 0, all = 0;
      for (int l = 0; l < min(kWave, a.c.n_seqs - seq); ++l) {
        const int c = __builtin_amdgcn_readlane(count, l);
        all += c;
        before += __builtin_amdgcn_readlane(order, l) > order ? c : 0;
      }
      if (tile >= all) {
        tile -= all;
        continue;
      }
      const int l = __builtin_ctzll(__builtin_amdgcn_ballot_w64(before <= tile && tile < before + count));
      tile -= __builtin_amdgcn_readlane(before, l);
      seq += l;
      s = Span{__builtin_amdgcn_readlane(mine.row0, l), __builtin_amdgcn_readlane(mine.past, l),
               __builtin_amdgcn_readlane(mine.n, l)};
      break;
    }
  }
  const int rows = s.n * a.group, r0 = tile * kCols;
  if (r0 >= rows) return;
  const int len = s.past + s.n;
  const int last_place = s.past + a.over(min(r0 + kCols, rows) - 1);
  const Visits visits(s.past + a.over(r0), last_place, a.window, a.sinks);
  const int begin = split * a.per, end = min(visits.count, begin + a.per);
  if (begin >= end) return;
  // the wavefront's columns; those behind the last row repeat it
  const int c0 = r0 + wide * kCol;
  const bool idle = c0 >= rows;
  const int lo_place = s.past + a.over(min(c0, rows - 1)), hi_place = s.past + a.over(min(c0 + kCol, rows) - 1);
  // the last visit is the open block, whose tokens are in the tail, where the workgroup's rows reach it
  const bool open = last_place / kBlock == len / kBlock;
  const int code_end = a.c.n_pages > 0 && !idle ? min(end, visits.count - (open ? 1 : 0)) : begin;

  const int row = min(c0 + col, rows - 1), row_token = a.over(row), place = s.past + row_token;
  half8 q[L::kFrags];
  {
    const uint16_t* p = a.q + (s.row0 + row_token) * a.q_tok + (head * a.group + row - row_token * a.group) * a.q_head;
#pragma unroll
    for (int f = 0; f < L::kFrags; ++f) q[f] = *reinterpret_cast<const half8*>(p + L::column(f, g));
  }
  Tile acc[L::kOuts], st[L::kTiles];
#pragma unroll
  for (int n = 0; n < L::kOuts; ++n) acc[n] = Tile(0.f);
  float ref = -__builtin_inff(), l = 0.f;
  // fp16: acc is in units of the last page's scale. Such scales lie between 2^-33 and 2^8, so the sums
  // stay inside fp32's range whatever follows; bfloat16's do not, and there each page's sums are scaled.
  float unit = 1.f;
  u32x4 kw[kLoads], vw[kLoads];
  // what one wavefront alone reads passes by the caches; the larger tiles' pages are read by their neighbours
  // too (12 conversations in tiles of 32 rows 82 us past the caches, 61 through them)
  auto load = [&](const u32x4* p) { return kCol == 16 ? __builtin_nontemporal_load(p) : *p; };
  auto load_k = [&](int page) __attribute__((always_inline)) {
    const u32x4* src = reinterpret_cast<const u32x4*>(
                           a.c.codes + (static_cast<int64_t>(page) * 2 * a.c.kv + head) * (kBlock * D)) +
                       L::key_lane(lane);
#pragma unroll
    for (int i = 0; i < kLoads; ++i) kw[i] = load(src + L::key_at(i));
  };
  auto load_v = [&](int page) __attribute__((always_inline)) {
    const u32x4* src = reinterpret_cast<const u32x4*>(
                           a.c.codes + ((static_cast<int64_t>(page) * 2 + 1) * a.c.kv + head) * (kBlock * D)) +
                       L::value_lane(lane);
#pragma unroll
    for (int i = 0; i < kLoads; ++i) vw[i] = load(src + L::value_at(i));
  };
  // Weights of a page's (or the tail's, times 2^-low) scores; the sums so far follow a new reference and unit.
  auto weigh = [&](float c, bool mask, int first, float ratio, float low) __attribute__((always_inline)) {
    c = fmaxf(c, 1e-37f);  // never 0: c times a hidden score's -inf is one
    if (mask) {
      // the lane's scores are those of the keys base + kStep (i / 4) + i % 4
      const int base = first + 4 * g, last = place - base;
#pragma unroll
      for (int i = 0; i < L::kLane; ++i) {
        const int key = L::kStep * (i / 4) + i % 4;
        st[i / L::kEach][i % L::kEach] = key <= last ? st[i / L::kEach][i % L::kEach] : -__builtin_inff();
      }
      if (a.window > 0) {
        // (wraps only where every key is behind the row's place and hidden already)
        const int from = static_cast<int>(static_cast<uint32_t>(last) - static_cast<uint32_t>(a.window));
        const int sinks = a.sinks - base;
#pragma unroll
        for (int i = 0; i < L::kLane; ++i) {
          const int key = L::kStep * (i / 4) + i % 4;
          const bool seen = (key > from) | (key < sinks);
          st[i / L::kEach][i % L::kEach] = seen ? st[i / L::kEach][i % L::kEach] : -__builtin_inff();
        }
      }
    }
    float top = st[0][0];
#pragma unroll
    for (int i = 1; i < L::kLane; ++i) top = fmaxf(top, st[i / L::kEach][i % L::kEach]);
    top = L::max_of(top) * c;
    if (__builtin_amdgcn_ballot_w64(top > ref + 8.f) || ratio != 1.f) {
      const float next = fmaxf(ref, top);
      // a row that has seen no key yet keeps -inf
      const float grow = next == -__builtin_inff() ? 1.f : __builtin_amdgcn_exp2f(ref - next);
      ref = next;
      l *= grow;
#pragma unroll
      for (int n = 0; n < L::kOuts; ++n)
#pragma unroll
        for (int e = 0; e < L::kEach; ++e) acc[n][e] *= grow * ratio;
    }
    const float base = ref == -__builtin_inff() ? 0.f : ref + low;  // its weights are exp2(-inf - 0) = 0
#pragma unroll
    for (int i = 0; i < L::kLane; ++i) {
      st[i / L::kEach][i % L::kEach] =
          __builtin_amdgcn_exp2f(__builtin_fmaf(st[i / L::kEach][i % L::kEach], c, -base));
    }
  };

  // The weights in fp16, whatever the operands' type (the values' codes are exact in it), and their sum. Tiles of
  // 16 rows wait for memory and take a second part of 11 bits, so that their outputs are those of weights in 32
  // bits but for the last rounding (error against 64 bits of 64 sequences' tokens 2.4e-4 with one part, 2.1e-4, the
  // output's rounding alone, with two; 34.4 -> 34.7 us). The larger ones keep one part (two: 44 -> 52 us for 512
  // rows over 8289 tokens) and the sum of the rounded weights, so a token that has nearly all of it keeps its
  // values exactly.
  constexpr bool kFine = kCol == 16;
  auto round = [&](half8 (&p)[L::kPs], half8 (&rest)[L::kPs]) __attribute__((always_inline)) {
#pragma unroll
    for (int u = 0; u < L::kPs; ++u)
#pragma unroll
      for (int e = 0; e < 8; e += 2) {
        const int i = 8 * u + e;
        const f32x2 x = {st[i / L::kEach][i % L::kEach], st[i / L::kEach][i % L::kEach + 1]};
        const half2_ w = __builtin_convertvector(x, half2_);
        p[u][e] = w.x;
        p[u][e + 1] = w.y;
        if constexpr (kFine) {
          rest[u][e] = static_cast<_Float16>(x[0] - static_cast<float>(w.x));
          rest[u][e + 1] = static_cast<_Float16>(x[1] - static_cast<float>(w.y));
          l += x[0];
          l += x[1];
        } else {
          l = __builtin_amdgcn_fdot2(w, half2_{static_cast<_Float16>(1.f), static_cast<_Float16>(1.f)}, l, false);
        }
      }
  };

  // 64 of the wavefront's pages at a time: lane l holds the l-th one's place and scales
  for (int base = begin + deep; base < code_end; base += kDeep * kWave) {
    const int mine = base + kDeep * lane;
    int page_l = -1;
    float ks_l = 1.f, vs_l = 1.f;
    if (mine < code_end) {
      if (alone && a.window == 0 && base == begin + deep)
        page_l = early < a.c.n_pages ? early : -1;
      else
        page_l = static_cast<int>(a.c.page(seq, visits.page(mine)));
      if (page_l >= 0) {
        ks_l = a.c.scales[static_cast<int64_t>(page_l) * 2 * a.c.kv + head];
        vs_l = a.c.scales[(static_cast<int64_t>(page_l) * 2 + 1) * a.c.kv + head] * T::kUnit;
      }
    }
    const int count = min((code_end - base + kDeep - 1) / kDeep, kWave);
    // what is no page is read as the pool's first one and seen by no row
    int page = __builtin_amdgcn_readlane(page_l, 0);
    load_k(max(page, 0));
    load_v(max(page, 0));
    auto step = [&](int i, auto more) __attribute__((always_inline)) {
      const float k_scale = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, ks_l), i));
      const float v_scale = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, vs_l), i));
      const int next = decltype(more)::value ? __builtin_amdgcn_readlane(page_l, i + 1) : 0;
      const int first = visits.page(base + kDeep * i) * kBlock;
#pragma unroll
      for (int t = 0; t < L::kTiles; ++t) st[t] = Tile(0.f);
#pragma unroll
      for (int f = 0; f < L::kFrags; ++f)
#pragma unroll
        for (int t = 0; t < L::kTiles; ++t) {
          const u32x4 w = kw[t * (L::kFrags / 2) + f / 2];
          st[t] = T::mfma(T::codes(f % 2 ? u32x2{w.z, w.w} : u32x2{w.x, w.y}), q[f], st[t]);
        }
      // the next page's keys are on their way while this one's weights and values are worked on, its
      // values during the next one's scores (the last page is a copy of its own without them: a
      // condition here would make every wait one for all loads)
      __builtin_amdgcn_sched_barrier(0);
      if constexpr (decltype(more)::value) load_k(max(next, 0));
      __builtin_amdgcn_sched_barrier(0);
      const bool all = page >= 0 && first + kBlock - 1 <= lo_place &&
                       (a.window == 0 || hi_place - first < a.window || first + kBlock <= a.sinks);
      weigh(a.scale_log2 * k_scale, !all, page >= 0 ? first : 0x7fff0000, kUnits ? unit * inverse(v_scale) : 1.f,
            0.f);
      if constexpr (kUnits) unit = v_scale;
      half8 p[L::kPs], rest[L::kPs];
      round(p, rest);
      if (page < 0) {
#pragma unroll
        for (int k = 0; k < kLoads; ++k) vw[k] = u32x4{0, 0, 0, 0};
      }
#pragma unroll
      for (int n = 0; n < L::kOuts; n += 2) {
        Tile o[2];
#pragma unroll
        for (int k = 0; k < 2; ++k) o[k] = kUnits ? acc[n + k] : Tile(0.f);
#pragma unroll
        for (int u = 0; u < L::kPs; ++u)
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            const half8 v = F16::codes(L::value_codes(vw, n + k, u));
            o[k] = F16::mfma(v, p[u], o[k]);
            if constexpr (kFine) o[k] = F16::mfma(v, rest[u], o[k]);
          }
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          if constexpr (kUnits) {
            acc[n + k] = o[k];
          } else {
#pragma unroll
            for (int e = 0; e < L::kEach; ++e) acc[n + k][e] = __builtin_fmaf(o[k][e], v_scale, acc[n + k][e]);
          }
        }
      }
      __builtin_amdgcn_sched_barrier(0);
      if constexpr (decltype(more)::value) load_v(max(next, 0));
      __builtin_amdgcn_sched_barrier(0);
      page = next;
    };
    for (int i = 0; i < count - 1; ++i) step(i, std::true_type{});
    step(count - 1, std::false_type{});
  }

  // the tail, by the wavefronts whose turn it is
  if (open && !idle && visits.count - 1 >= begin && visits.count - 1 < end &&
      (visits.count - 1 - begin) % kDeep == deep) {
    const uint16_t* tk = a.c.tail + (static_cast<int64_t>(seq) * 2 * a.c.kv + head) * (kBlock * D);
    const uint16_t* tv = tk + static_cast<int64_t>(a.c.kv) * (kBlock * D);
    const int first = len / kBlock * kBlock, left = len - first;
#pragma unroll
    for (int t = 0; t < L::kTiles; ++t) {
      st[t] = Tile(0.f);
#pragma unroll
      for (int f = 0; f < L::kFrags; ++f)
        st[t] = T::mfma(*reinterpret_cast<const half8*>(tk + (t * kCol + col) * D + L::column(f, g)), q[f], st[t]);
    }
    weigh(a.scale_log2, true, first, unit, kUnits ? 0.f : 40.f);
    unit = 1.f;
    // the weights in the tail's type; for bfloat16 as two parts, so that they keep 16 bits
    half8 hi[L::kPs], lo[L::kPs];
    if constexpr (kUnits) {
      round(hi, lo);
    } else {
      float sum = 0.f;
#pragma unroll
      for (int i = 0; i < L::kLane; ++i) {
        const float x = st[i / L::kEach][i % L::kEach];
        const uint16_t b = T::down(x);
        hi[i / 8][i % 8] = __builtin_bit_cast(_Float16, b);
        lo[i / 8][i % 8] = __builtin_bit_cast(_Float16, T::down(x - T::up(b)));
        sum += x;
      }
      l += sum * (1.f / T::kUnit);
    }
#pragma unroll
    for (int n = 0; n < L::kOuts; ++n)
#pragma unroll
      for (int u = 0; u < L::kPs; ++u) {
        uint64_t w[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          // what lies behind the sequence's tokens is no value
          const int t = L::kStep * (2 * u + e) + g * 4, there = min(max(left - t, 0), 4);
          w[e] = *reinterpret_cast<const uint64_t*>(tv + (n * kCol + col) * kBlock + t);
          w[e] &= there == 4 ? ~uint64_t{0} : (uint64_t{1} << (16 * there)) - 1;
        }
        struct Two { uint64_t x, y; };
        const half8 v = __builtin_bit_cast(half8, Two{w[0], w[1]});
        acc[n] = T::mfma(v, hi[u], acc[n]);
        if constexpr (!kUnits || kFine) acc[n] = T::mfma(v, lo[u], acc[n]);
      }
  }

  // The wavefronts' sums to one reference, and where there is no other part over the sum of the weights; a
  // row's columns are then only added up.
  const bool only = visits.count <= a.per;
  constexpr int kFours = L::kEach / 4;
  l = L::sum_of(l);
  const int mine = wide * kCol + col;
  if (g == 0) {
    stat[0][deep][mine] = ref;
    stat[1][deep][mine] = l;
  }
  __syncthreads();
  float top = stat[0][0][mine], sum = 0.f;
#pragma unroll
  for (int w = 1; w < kDeep; ++w) top = fmaxf(top, stat[0][w][mine]);
#pragma unroll
  for (int w = 0; w < kDeep; ++w) {
    const float x = stat[0][w][mine];
    sum += x == -__builtin_inff() ? 0.f : stat[1][w][mine] * __builtin_amdgcn_exp2f(x - top);
  }
  float by = ref == -__builtin_inff() ? 0.f : __builtin_amdgcn_exp2f(ref - top) * unit;
  if (only) by *= sum > 0.f ? 1.f / sum : sum == 0.f ? 0.f : sum;  // a sum that is NaN stays one
#pragma unroll
  for (int i = 0; i < L::kOuts * kFours; ++i) {
    const Tile& o = acc[i / kFours];
    const int e = i % kFours * 4;
    *reinterpret_cast<f32x4*>(&part[deep][mine][kCol == 16 ? i * 16 + g * 4 : i * 8 + g * 4]) =
        f32x4{o[e] * by, o[e + 1] * by, o[e + 2] * by, o[e + 3] * by};
  }
  __syncthreads();
  if (!only && deep == 0 && g == 0 && r0 + mine < rows) {
    const int token = a.over(r0 + mine);
    const int64_t to = static_cast<int64_t>(s.row0 + token) * a.n_q + head * a.group + r0 + mine - token * a.group;
    a.part_ml[to * a.splits + split] = make_float2(top, sum);
  }
#pragma unroll
  for (int i = 0; i < kCols * D / 4 / kThreads; ++i) {
    const int c = (i * kThreads + tid) / (D / 4), d = tid % (D / 4) * 4, r = r0 + c, token = a.over(r);
    const int64_t to = static_cast<int64_t>(s.row0 + token) * a.n_q + head * a.group + r - token * a.group;
    f32x4 o = *reinterpret_cast<const f32x4*>(&part[0][c][d]);
#pragma unroll
    for (int w = 1; w < kDeep; ++w) {
      const f32x4 y = *reinterpret_cast<const f32x4*>(&part[w][c][d]);
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] += y[e];
    }
    if (r >= rows) continue;
    if (only) {
      *reinterpret_cast<u32x2*>(a.out + to * D + d) = outputs<T>(o);
    } else {
      *reinterpret_cast<f32x4*>(a.part_o + (to * a.splits + split) * D + d) = o;
    }
  }
}

// Sum and maximum over a wavefront in every lane, through VALU operands.
__device__ __forceinline__ float lanes_max(float x) {
  return __builtin_bit_cast(float, lanes_reduce(__builtin_bit_cast(uint32_t, x), [](uint32_t p, uint32_t q) {
    return __builtin_bit_cast(uint32_t, fmaxf(__builtin_bit_cast(float, p), __builtin_bit_cast(float, q)));
  }));
}
__device__ __forceinline__ float lanes_sum(float x) {
  return __builtin_bit_cast(float, lanes_reduce(__builtin_bit_cast(uint32_t, x), [](uint32_t p, uint32_t q) {
    return __builtin_bit_cast(uint32_t, __builtin_bit_cast(float, p) + __builtin_bit_cast(float, q));
  }));
}

// The parts of a row and head, joined in their order. kRows = 0: a workgroup has 32 columns of one, its
// 32 groups of 8 threads take every 32nd part (up to 256). Else a wavefront has all D columns of kRows of
// them, its groups of D / 4 lanes take every second part (fourth with 64 columns), kEach each. All loads are
// on their way before the weights are known. 3 to 4 us, a launch's least and two misses, for one token's 16
// or 256 parts as for 64 sequences' 13 each; 16 MB of a long piece's parts 5.8.
template <class T, int D, int kRows, int kEach>
__global__ __launch_bounds__(kThreads) void cache_join_kernel(AttnArgs a) {
  constexpr bool kWide = kRows == 0;
  constexpr int kLanes = kWide ? 8 : D / 4, kGroups = (kWide ? kThreads : kWave) / kLanes, kR = kWide ? 1 : kRows;
  constexpr int kSlices = kWide ? D / 32 : 1, kPer = kWide ? kSplits / kWave : 1;
  __shared__ float weight[kWide ? kSplits : 1];
  __shared__ f32x4 sums[kWide ? kGroups : 1][kLanes];
  const int lane = threadIdx.x & 63, tid = kWide ? threadIdx.x : lane;
  uint32_t item = kWide ? blockIdx.x : blockIdx.x * kWaves + __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int slice = static_cast<int>(item % kSlices);
  item = item / kSlices * kR;
  const int grp = tid / kLanes, d = slice * 4 * kLanes + (tid % kLanes) * 4;
  int seq, at, qh;
  {
    const uint32_t rest = item / a.n_q;
    qh = static_cast<int>(item - rest * a.n_q);
    seq = static_cast<int>(rest / a.max_new);
    at = static_cast<int>(rest) - seq * a.max_new;
  }
  int64_t to[kR];
  int parts[kR];
#pragma unroll
  for (int k = 0; k < kR; ++k) {
    to[k] = parts[k] = 0;
    if (seq < a.c.n_seqs) {
      const Span s = span_of(a.bounds, a.past, seq, a.n_rows, a.max_new, a.max_len);
      if (at < s.n) {
        const int rows = s.n * a.group, r0 = (at * a.group + qh - a.over(qh) * a.group) & ~(a.cols - 1);
        const Visits visits(s.past + a.over(r0), s.past + a.over(min(r0 + a.cols, rows) - 1), a.window, a.sinks);
        parts[k] = (visits.count + a.per - 1) / a.per;
        to[k] = static_cast<int64_t>(s.row0 + at) * a.n_q + qh;
      }
    }
    if (++qh == a.n_q) {
      qh = 0;
      if (++at == a.max_new) {
        at = 0;
        ++seq;
      }
    }
  }
  f32x4 o[kR][kEach];
  float2 ml[kR][kPer];
#pragma unroll
  for (int k = 0; k < kR; ++k) {
    if (parts[k] <= 1) continue;  // nothing, or written by its one part
    const float* p = a.part_o + to[k] * a.splits * D + d;
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      const int j = grp + i * kGroups;
      o[k][i] = f32x4{0.f, 0.f, 0.f, 0.f};
      if (j < parts[k]) o[k][i] = *reinterpret_cast<const f32x4*>(p + static_cast<int64_t>(j) * D);
    }
    // every wavefront takes all weights
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int j = lane + i * kWave;
      ml[k][i] = j < parts[k] ? a.part_ml[to[k] * a.splits + j] : make_float2(-__builtin_inff(), 0.f);
    }
  }
#pragma unroll
  for (int k = 0; k < kR; ++k) {
    if (parts[k] <= 1) continue;
    float top = -__builtin_inff(), w[kPer], sum = 0.f;
#pragma unroll
    for (int i = 0; i < kPer; ++i) top = fmaxf(top, ml[k][i].x);
    top = lanes_max(top);
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      w[i] = ml[k][i].x == -__builtin_inff() ? 0.f : __builtin_amdgcn_exp2f(ml[k][i].x - top);
      sum += ml[k][i].y * w[i];
    }
    sum = lanes_sum(sum);
    f32x4 total = {0.f, 0.f, 0.f, 0.f};
    if constexpr (kWide) {
      if (threadIdx.x < kWave) {
#pragma unroll
        for (int i = 0; i < kPer; ++i) weight[lane + i * kWave] = w[i];
      }
      __syncthreads();
    }
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      const int j = grp + i * kGroups;
      const float by = kWide ? weight[kWide ? j : 0] : __shfl(w[0], j & 63, kWave);
      if (j < parts[k]) {
#pragma unroll
        for (int e = 0; e < 4; ++e) total[e] += by * o[k][i][e];
      }
    }
    if constexpr (kWide) {
      sums[grp][tid % kLanes] = total;
      __syncthreads();
      if (grp != 0) return;
      const int used = min(kGroups, parts[k]);
      for (int i = 1; i < used; ++i) {
        const f32x4 x = sums[i][tid];
#pragma unroll
        for (int e = 0; e < 4; ++e) total[e] += x[e];
      }
    } else {
#pragma unroll
      for (int off = kLanes; off < kWave; off *= 2)
#pragma unroll
        for (int e = 0; e < 4; ++e) total[e] += __shfl_xor(total[e], off, kWave);
    }
    if (grp == 0) {
      const float inv = sum > 0.f ? 1.f / sum : sum == 0.f ? 0.f : sum;
#pragma unroll
      for (int e = 0; e < 4; ++e) total[e] *= inv;
      *reinterpret_cast<u32x2*>(a.out + to[k] * D + d) = outputs<T>(total);
    }
  }
}

// How an attention call is cut: rows of a tile, tiles of a KV head at most, parts of the pages and pages of
// a part.
struct Plan {
  int wide;  // 0: 16 rows a workgroup, one tile a sequence; 1, 2: kWide of 32 each
  int64_t cols, tiles, splits, per;
};
Plan plan_with(int wide, int64_t n_rows, int64_t n_seqs, int64_t kv, int64_t group, int64_t max_new, int64_t max_len,
               int64_t window, int64_t sinks) {
  Plan p;
  sinks = std::min(sinks, max_len);
  p.wide = wide;
  p.cols = wide ? 32 * wide : 16;
  // a sequence's last tile may be part of one; no more rows than there are
  p.tiles = n_seqs;
  if (wide) {
    const int64_t rows = max_new * group, near = kNear;
    p.tiles = std::min(n_seqs * ((rows + p.cols - 1) / p.cols), (n_rows * group + p.cols - 1) / p.cols + n_seqs);
    p.tiles = (p.tiles + near - 1) / near * near;
  }
  int64_t visits = (max_len + kBlock - 1) / kBlock;
  if (window > 0)
    visits = std::min(visits, (window + p.cols - 1 + kBlock - 1) / kBlock + 1 + (sinks + kBlock - 1) / kBlock);
  // Parts cost their join: a launch, and 520 bytes a row written and read again. Two workgroups a CU, parts of
  // at least a page per wavefront. No parts where one's pages in turn take no longer than the join: 16 pages,
  // 32 where 16-row tiles fill half of the CUs, 48 where larger ones fill a quarter (one token of 64
  // sequences over 1001 and 2001 tokens 16.5 and 20.8 us in parts, 10.6 and 16.2 without; of 128 over 2001
  // 34.6 and 29). Else 16-row tiles have short parts where there are few sequences, since those of other
  // lengths than the longest leave CUs idle at the end (64 sequences of 201 to 8191: 36 us in parts of 10
  // pages, 40 in 32), and long ones where there are many (256 over 2001: 64 in 10, 51 in 32). All within
  // 8192 workgroups (a part that a sequence lacks costs a start) and 128 MB of parts.
  const int64_t cus = device_cus(), base = std::max<int64_t>(kv * p.tiles, 1);
  const int64_t most = std::min<int64_t>({kSplits, 8192 / base, (int64_t{1} << 27) / (n_rows * kv * group * 520 + 1)});
  const bool filled = base >= (wide ? cus / 4 : cus / 2);
  int64_t want = 2 * cus / base;
  if (visits <= (!filled ? 16 : wide ? 48 : 32)) {
    want = 1;
  } else if (!wide) {
    const int64_t pages = base < cus ? 10 : base < 2 * cus ? 32 : 64;
    want = std::max(want, (visits + pages - 1) / pages);
  }
  want = std::max<int64_t>(1, std::min(want, most));
  p.per = std::max<int64_t>((visits + want - 1) / want, kWaves);
  p.splits = std::max<int64_t>((visits + p.per - 1) / p.per, 1);
  return p;
}
// Tiles of 64 rows or of 32, whichever end first: a round of the workgroups takes as long as some 4 pages and
// its wavefronts' pages, parts and their join 6 (one text's 512 rows over 8289 tokens 48 us in tiles of 64, 52
// in 32; 1000 rows over 9000 90 and 83, 190 over 1334 17.0 and 14.5; 12 texts of 200 to 4000 tokens, 10 to 150
// rows each, 54 and 45).
Plan plan_of(int64_t n_rows, int64_t n_seqs, int64_t kv, int64_t group, int64_t max_new, int64_t max_len,
             int64_t window, int64_t sinks) {
  auto with = [&](int wide) { return plan_with(wide, n_rows, n_seqs, kv, group, max_new, max_len, window, sinks); };
  const int64_t rows = max_new * group;
  if (rows <= 32) return with(rows <= 16 ? 0 : 1);
  auto cost = [&](const Plan& p) {
    const int64_t deep = kWaves / p.wide;
    const double rounds = std::max(1.0, static_cast<double>(kv * p.tiles * p.splits) / (2.0 * device_cus()));
    return rounds * static_cast<double>(4 + (p.per + deep - 1) / deep) + (p.splits > 1 ? 6.0 : 0.0);
  };
  const Plan one = with(1), two = with(2);
  return cost(two) < cost(one) ? two : one;
}

bool cache_shape(int32_t n_kv, int32_t head_dim, int32_t dtype, int32_t n_seqs, int64_t n_pages, int32_t width,
                 int64_t n_rows) {
  return n_kv >= 1 && n_kv <= 1024 && (head_dim == 64 || head_dim == 128) &&
         (dtype == TALM_F16 || dtype == TALM_BF16) && n_seqs >= 0 && n_seqs <= (1 << 24) && n_pages >= 0 &&
         n_pages < (int64_t{1} << 31) && width >= 0 && width <= (1 << 24) && n_rows >= 0 && n_rows < (int64_t{1} << 31);
}

bool strides_fit(int64_t tok, int64_t head) { return tok % 8 == 0 && head % 8 == 0 && tok >= 0 && head >= 0; }

}  // namespace
}  // namespace talm

using namespace talm;

#define TALM_CACHE_KERNEL(name, grid, args)                                                                   \
  do {                                                                                                        \
    const dim3 g_(grid), b_(kThreads);                                                                        \
    if (dtype == TALM_F16 && head_dim == 128) name(F16, 128, g_, b_, args);                                   \
    else if (dtype == TALM_F16) name(F16, 64, g_, b_, args);                                                  \
    else if (head_dim == 128) name(BF16, 128, g_, b_, args);                                                  \
    else name(BF16, 64, g_, b_, args);                                                                        \
  } while (0)

TALM_API int talm_cache_write(const uint16_t* k, int64_t k_stride_tok, int64_t k_stride_head, const uint16_t* v,
                              int64_t v_stride_tok, int64_t v_stride_head, int64_t n_rows, int32_t n_kv_heads,
                              int32_t head_dim, int32_t dtype, const int32_t* bounds, const int32_t* past,
                              int32_t n_seqs, int32_t max_new, uint8_t* codes, float* scales, uint16_t* tail,
                              const int32_t* table, int64_t n_pages, int32_t width, const float* cos,
                              const float* sin, int64_t cs_stride, const uint16_t* q, int64_t q_stride_tok,
                              int64_t q_stride_head, int32_t n_q_heads, uint16_t* q_out, void* stream) {
  if (!cache_shape(n_kv_heads, head_dim, dtype, n_seqs, n_pages, width, n_rows) || max_new < 0 || n_q_heads < 0)
    return fail(TALM_EINVAL, "cache_write: bad shape rows=%lld sequences=%d kv=%d head_dim=%d (64, 128) dtype=%d",
                (long long)n_rows, n_seqs, n_kv_heads, head_dim, dtype);
  const bool turn = cos != nullptr;
  if (turn != (sin != nullptr) || (!turn && n_q_heads) || (turn && (cs_stride < head_dim || cs_stride % 4)))
    return fail(TALM_EINVAL, "cache_write: cos and sin both or neither, of rows of at least head_dim, a multiple of 4; "
                "queries only with them");
  if (n_rows == 0) return ok();
  const bool some = n_seqs && width && max_new;  // else nothing is put into the cache
  if ((some && (!k || !v || !bounds || !past || !tail || !table || (n_pages && (!scales || !codes)))) ||
      (n_q_heads && (!q || !q_out)))
    return fail(TALM_EINVAL, "cache_write: null pointer");
  if (!strides_fit(k_stride_tok, k_stride_head) || !strides_fit(v_stride_tok, v_stride_head) ||
      (n_q_heads && !strides_fit(q_stride_tok, q_stride_head)))
    return fail(TALM_EINVAL, "cache_write: strides must be multiples of 8");
  for (const void* p : {static_cast<const void*>(k), static_cast<const void*>(v), static_cast<const void*>(codes),
                        static_cast<const void*>(tail), static_cast<const void*>(cos), static_cast<const void*>(sin),
                        static_cast<const void*>(n_q_heads ? q : nullptr), static_cast<const void*>(q_out)})
    if (!aligned(p, 16)) return fail(TALM_EINVAL, "cache_write: buffers must be 16-byte aligned");
  max_new = static_cast<int32_t>(std::min<int64_t>(max_new, n_rows));
  WriteArgs a{k, k_stride_tok, k_stride_head, v, v_stride_tok, v_stride_head, n_rows, bounds, past, max_new,
              width * kBlock, (max_new + kBlock - 1) / kBlock + 1, codes, scales, tail,
              Cache{codes, scales, tail, table, n_pages, width, n_seqs, n_kv_heads}, cos, sin, cs_stride, q,
              q_stride_tok, q_stride_head, n_q_heads, q_out, 0, 0};
  a.kv_items = some ? static_cast<int64_t>(n_seqs) * n_kv_heads * 2 * a.chunks : 0;
  const int64_t turns = turn ? (n_rows * n_q_heads * (head_dim / 8) + kThreads - 1) / kThreads : 0;
  if (a.kv_items + turns > 0x7fffffff) return fail(TALM_EINVAL, "cache_write: too many tokens");
  if (a.kv_items + turns == 0) return ok();
  const hipStream_t st = as_stream(stream);
#define LAUNCH(T, D, grid, block, args)                                                     \
  do {                                                                                      \
    if (turn)                                                                               \
      hipLaunchKernelGGL((cache_write_kernel<T, D, true>), grid, block, 0, st, args);       \
    else                                                                                    \
      hipLaunchKernelGGL((cache_write_kernel<T, D, false>), grid, block, 0, st, args);      \
  } while (0)
  for (int64_t first = 0; first < a.kv_items + turns; first += kGrid) {
    a.first = static_cast<uint32_t>(first);
    TALM_CACHE_KERNEL(LAUNCH, static_cast<unsigned>(std::min(a.kv_items + turns - first, kGrid)), a);
    if (const int status = check_launch("cache_write")) return status;
  }
#undef LAUNCH
  return ok();
}

TALM_API int talm_cache_read(const uint8_t* codes, const float* scales, const uint16_t* tail, const int32_t* table,
                             int64_t n_pages, int32_t width, int32_t n_seqs, int32_t n_kv_heads, int32_t head_dim,
                             int32_t dtype, const int32_t* length, const int32_t* bounds, const int32_t* past,
                             int32_t max_new, int64_t n_rows, uint16_t* k, uint16_t* v, void* stream) {
  if (!cache_shape(n_kv_heads, head_dim, dtype, n_seqs, n_pages, width, n_rows) || max_new < 0)
    return fail(TALM_EINVAL, "cache_read: bad shape rows=%lld sequences=%d kv=%d head_dim=%d (64, 128) dtype=%d",
                (long long)n_rows, n_seqs, n_kv_heads, head_dim, dtype);
  if (n_rows == 0 || n_seqs == 0 || max_new == 0 || width == 0) return ok();
  if ((n_pages && (!codes || !scales)) || !tail || !table || !length || !bounds || !past || !k || !v)
    return fail(TALM_EINVAL, "cache_read: null pointer");
  for (const void* p : {static_cast<const void*>(codes), static_cast<const void*>(tail), static_cast<const void*>(k),
                        static_cast<const void*>(v)})
    if (!aligned(p, 16)) return fail(TALM_EINVAL, "cache_read: buffers must be 16-byte aligned");
  max_new = static_cast<int32_t>(std::min<int64_t>(max_new, n_rows));
  ReadArgs a{Cache{codes, scales, tail, table, n_pages, width, n_seqs, n_kv_heads}, length, bounds, past, n_rows,
                   max_new, width * kBlock, (max_new + kBlock - 1) / kBlock + 1, k, v, 0};
  const int64_t items = static_cast<int64_t>(n_seqs) * n_kv_heads * 2 * a.chunks;
  if (items > 0x7fffffff) return fail(TALM_EINVAL, "cache_read: too many tokens");
  const hipStream_t st = as_stream(stream);
#define LAUNCH(T, D, grid, block, args) hipLaunchKernelGGL((cache_read_kernel<T, D>), grid, block, 0, st, args)
  for (int64_t first = 0; first < items; first += kGrid) {
    a.first = static_cast<uint32_t>(first);
    TALM_CACHE_KERNEL(LAUNCH, static_cast<unsigned>(std::min(items - first, kGrid)), a);
    if (const int status = check_launch("cache_read")) return status;
  }
#undef LAUNCH
  return ok();
}

namespace {
bool attn_shape(int64_t n_rows, int32_t n_q, int32_t n_kv, int32_t head_dim, int32_t n_seqs, int32_t max_new,
                int32_t max_len, int32_t window, int32_t sinks) {
  return n_kv >= 1 && n_kv <= 1024 && n_q >= 1 && n_q <= 65536 && n_q % n_kv == 0 &&
         (head_dim == 64 || head_dim == 128) && n_rows >= 0 && n_rows < (int64_t{1} << 31) && n_seqs >= 0 &&
         max_new >= 0 && static_cast<int64_t>(max_new) * (n_q / n_kv) < (int64_t{1} << 30) && max_len >= 0 &&
         max_len <= (1 << 30) && window >= 0 && sinks >= 0;
}
}  // namespace

TALM_API int64_t talm_cache_attn_workspace(int64_t n_rows, int32_t n_q_heads, int32_t n_kv_heads, int32_t head_dim,
                                           int32_t n_seqs, int32_t max_new, int32_t max_len, int32_t window,
                                           int32_t sinks) {
  if (!attn_shape(n_rows, n_q_heads, n_kv_heads, head_dim, n_seqs, max_new, max_len, window, sinks)) return -1;
  max_new = static_cast<int32_t>(std::min<int64_t>(max_new, n_rows));
  const Plan p = plan_of(n_rows, n_seqs, n_kv_heads, n_q_heads / n_kv_heads, max_new, max_len, window, sinks);
  return p.splits > 1 ? n_rows * n_q_heads * p.splits * (head_dim + 2) * static_cast<int64_t>(sizeof(float)) : 0;
}

TALM_API int talm_cache_attn(const uint16_t* q, int64_t q_stride_tok, int64_t q_stride_head, int64_t n_rows,
                             int32_t n_q_heads, int32_t n_kv_heads, int32_t head_dim, int32_t dtype,
                             const int32_t* bounds, const int32_t* past, int32_t n_seqs, int32_t max_new,
                             int32_t max_len, const uint8_t* codes, const float* scales, const uint16_t* tail,
                             const int32_t* table, int64_t n_pages, int32_t width, float scale, int32_t window,
                             int32_t sinks, uint16_t* out, void* workspace, int64_t workspace_bytes, void* stream) {
  if (!cache_shape(n_kv_heads, head_dim, dtype, n_seqs, n_pages, width, n_rows) ||
      !attn_shape(n_rows, n_q_heads, n_kv_heads, head_dim, n_seqs, max_new, max_len, window, sinks))
    return fail(TALM_EINVAL, "cache_attn: bad shape rows=%lld sequences=%d heads=%d/%d head_dim=%d (64, 128) dtype=%d "
                "max_new=%d max_len=%d window=%d sinks=%d", (long long)n_rows, n_seqs, n_q_heads, n_kv_heads, head_dim,
                dtype, max_new, max_len, window, sinks);
  if (!(scale > 0.f) || !(scale < INFINITY)) return fail(TALM_EINVAL, "cache_attn: scale must be positive and finite");
  if (n_rows == 0 || n_seqs == 0 || max_new == 0 || max_len == 0 || width == 0) return ok();
  if (!q || !bounds || !past || (n_pages && (!codes || !scales)) || !tail || !table || !out)
    return fail(TALM_EINVAL, "cache_attn: null pointer");
  if (!strides_fit(q_stride_tok, q_stride_head)) return fail(TALM_EINVAL, "cache_attn: strides must be multiples of 8");
  for (const void* p : {static_cast<const void*>(q), static_cast<const void*>(codes), static_cast<const void*>(tail),
                        static_cast<const void*>(out), static_cast<const void*>(workspace)})
    if (!aligned(p, 16)) return fail(TALM_EINVAL, "cache_attn: buffers must be 16-byte aligned");
  const int64_t need = talm_cache_attn_workspace(n_rows, n_q_heads, n_kv_heads, head_dim, n_seqs, max_new, max_len,
                                                 window, sinks);
  if (workspace_bytes < need || (need && !workspace))
    return fail(TALM_EINVAL, "cache_attn: workspace of %lld bytes, %lld needed", (long long)workspace_bytes,
                (long long)need);
  max_new = static_cast<int32_t>(std::min<int64_t>(max_new, n_rows));
  const Plan p = plan_of(n_rows, n_seqs, n_kv_heads, n_q_heads / n_kv_heads, max_new, max_len, window, sinks);
  float* part_o = static_cast<float*>(workspace);
  // n / group for n < 2^30 as (n magic) >> e, magic = ceil(2^e / group), e = 30 + ceil(log2 group), both
  // shifted up to a product's upper half (group is at most 2^16, so magic is below 2^32)
  const int64_t group = n_q_heads / n_kv_heads;
  int e = 30;
  while ((int64_t{1} << (e - 30)) < group) ++e;
  uint64_t magic = ((uint64_t{1} << e) + group - 1) / group;
  while (e < 32) {
    magic <<= 1;
    ++e;
  }
  AttnArgs a{Cache{codes, scales, tail, table, n_pages, width, n_seqs, n_kv_heads}, bounds, past,
             static_cast<int>(n_rows), max_new, std::min(max_len, width * kBlock), n_q_heads, static_cast<int>(group),
             static_cast<int>(static_cast<uint32_t>(magic)), e - 32, static_cast<int>(p.cols),
             static_cast<int>(p.splits), static_cast<int>(p.per),
             p.splits >= 8 ? 7 : p.splits >= 4 ? 3 : p.splits >= 2 ? 1 : 0, p.wide != 0, window,
             std::min(sinks, max_len), scale * 1.44269504088896340736f, q, q_stride_tok, q_stride_head, out, part_o,
             reinterpret_cast<float2*>(part_o ? part_o + n_rows * n_q_heads * p.splits * head_dim : nullptr)};
  const int64_t items = (p.wide ? p.tiles : 1) * p.splits;
  const int64_t joins = p.splits > 1 ? static_cast<int64_t>(n_seqs) * max_new * n_q_heads : 0;
  // groups of D / 4 lanes in a wavefront; one row's few parts are too little work for it
  const int lanes = kWave * 4 / head_dim;
  const int rows = p.splits <= 2 * lanes ? 4 : p.splits <= 8 * lanes ? 1 : 0;
  const int64_t groups = rows ? (joins + rows * kWaves - 1) / (rows * kWaves) : joins * (head_dim / 32);
  if (items > kGrid || joins > 0x7fffffff || groups > kGrid || (!p.wide && n_seqs > 65535))
    return fail(TALM_EINVAL, "cache_attn: too many rows, or more than 65535 sequences of few");
  const hipStream_t st = as_stream(stream);
#define LAUNCH(T, D, grid, block, args)                                                    \
  do {                                                                                     \
    if (p.wide == 0)                                                                       \
      hipLaunchKernelGGL((cache_attn_kernel<T, D, 16, 1>), grid, block, 0, st, args);       \
    else if (p.wide == 1)                                                                  \
      hipLaunchKernelGGL((cache_attn_kernel<T, D, 32, 1>), grid, block, 0, st, args);       \
    else                                                                                   \
      hipLaunchKernelGGL((cache_attn_kernel<T, D, 32, 2>), grid, block, 0, st, args);       \
  } while (0)
  TALM_CACHE_KERNEL(LAUNCH, dim3(static_cast<unsigned>(items), n_kv_heads, p.wide ? 1 : n_seqs), a);
#undef LAUNCH
  if (const int status = check_launch("cache_attn")) return status;
  if (joins == 0) return TALM_OK;
#define LAUNCH(T, D, grid, block, args)                                                   \
  do {                                                                                    \
    if (rows == 4)                                                                        \
      hipLaunchKernelGGL((cache_join_kernel<T, D, 4, 2>), grid, block, 0, st, args);      \
    else if (rows == 1)                                                                   \
      hipLaunchKernelGGL((cache_join_kernel<T, D, 1, 8>), grid, block, 0, st, args);      \
    else                                                                                  \
      hipLaunchKernelGGL((cache_join_kernel<T, D, 0, 8>), grid, block, 0, st, args);      \
  } while (0)
  TALM_CACHE_KERNEL(LAUNCH, static_cast<unsigned>(groups), a);
#undef LAUNCH
  return check_launch("cache_attn");
}
