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
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

constexpr int kBlock = 64;     // tokens of a page
constexpr int kThreads = 256;
constexpr int kWaves = kThreads / kWave;
constexpr int kSplits = 256;   // the most parts that the keys of a row are split into

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
  int64_t row0;
  int past, n;
};
__device__ __forceinline__ Span span_of(const int32_t* bounds, const int32_t* past, int seq, int64_t n_rows,
                                        int max_new, int max_len) {
  const int64_t lo = max(int64_t{0}, min(static_cast<int64_t>(bounds[2 * seq]), n_rows));
  const int64_t hi = max(lo, min(static_cast<int64_t>(bounds[2 * seq + 1]), n_rows));
  Span s{lo, past[seq], static_cast<int>(min(hi - lo, static_cast<int64_t>(max_new)))};
  if (s.past < 0 || s.past >= max_len) return Span{lo, 0, 0};
  s.n = min(s.n, max_len - s.past);
  return s;
}

struct F16 {
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
};
struct BF16 {
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
// stores the tokens behind the last complete block into it, so no other touches the tail.
template <class T, int D, bool kTurn>
__global__ __launch_bounds__(kThreads) void cache_write_kernel(WriteArgs a) {
  constexpr int kPer = D / 8;  // 16-byte pieces of a row
  __shared__ alignas(16) uint16_t tile[kBlock][D + 2];
  __shared__ float tops[kWaves];
  const int tid = threadIdx.x, lane = tid & 63;
  if (kTurn && blockIdx.x >= a.kv_items) {
    const int64_t i = (blockIdx.x - a.kv_items) * kThreads + tid;
    if (i >= a.n_rows * a.n_q * kPer) return;
    const int d = static_cast<int>(i % kPer) * 8;
    const int64_t rh = i / kPer, row = rh / a.n_q;
    const int head = static_cast<int>(rh - row * a.n_q);
    uint32_t w[4];
    row8<T, D>(a.q + row * a.q_tok + head * a.q_head, a.cos + row * a.cs_tok, a.sin + row * a.cs_tok, d, true, w);
    *reinterpret_cast<u32x4*>(a.q_out + rh * D + d) = u32x4{w[0], w[1], w[2], w[3]};
    return;
  }
  const int j = static_cast<int>(blockIdx.x % a.chunks);
  const int rest = static_cast<int>(blockIdx.x / a.chunks);
  const int which = rest & 1, head = (rest >> 1) % a.c.kv, seq = (rest >> 1) / a.c.kv;
  const Span s = span_of(a.bounds, a.past, seq, a.n_rows, a.max_new, a.max_len);
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
    const int64_t row = s.row0 + (t - s.past);
    row8<T, D>(src + row * tok, kTurn ? a.cos + row * a.cs_tok : nullptr, kTurn ? a.sin + row * a.cs_tok : nullptr,
               d, turn, w);
  };
  if (block < last) {
    const int64_t page = a.c.page(seq, block);
    // the block to LDS: pieces of 8 columns, a row's behind each other
    float top = 0.f;
    for (int i = tid; i < kBlock * kPer; i += kThreads) {
      const int t = i / kPer, d = (i % kPer) * 8, at = block * kBlock + t;
      uint32_t w[4];
      if (at < s.past) {
        if (which == 0) {
          const u32x4 x = *reinterpret_cast<const u32x4*>(tail + t * D + d);
#pragma unroll
          for (int e = 0; e < 4; ++e) w[e] = x[e];
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            w[e] = tail[(d + 2 * e) * kBlock + t] |
                   static_cast<uint32_t>(tail[(d + 2 * e + 1) * kBlock + t]) << 16;
        }
      } else {
        fresh(at, d, w);
      }
      top = top_of<T>(w, top);
#pragma unroll
      for (int e = 0; e < 4; ++e) *reinterpret_cast<uint32_t*>(&tile[t][d + 2 * e]) = w[e];
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
};

// code * scale in 16 bits. In fp16 a value just under 65504 may have been rounded up to 65536, which
// the type does not hold: its largest number stands for it.
template <class T>
__device__ __forceinline__ uint16_t held(float code, float scale) {
  float x = code * scale;
  if constexpr (__is_same(T, F16)) {
    if (fabsf(x) > 65504.f) x = copysignf(65504.f, x);
  }
  return T::down(x);
}

// One workgroup: one block of one sequence, one KV head, keys or values.
template <class T, int D>
__global__ __launch_bounds__(kThreads) void cache_read_kernel(ReadArgs a) {
  constexpr int kPer = D / 8;
  __shared__ alignas(16) uint16_t tile[kBlock][D + 2];
  const int tid = threadIdx.x;
  const int j = static_cast<int>(blockIdx.x % a.chunks);
  const int rest = static_cast<int>(blockIdx.x / a.chunks);
  const int which = rest & 1, head = (rest >> 1) % a.c.kv, seq = (rest >> 1) / a.c.kv;
  const Span s = span_of(a.bounds, a.past, seq, a.n_rows, a.max_new, a.max_len);
  const int len = min(max(a.length[seq], 0), a.max_len);
  const int block = s.past / kBlock + j;
  const int lo = max(block * kBlock, s.past), hi = min((block + 1) * kBlock, s.past + s.n);
  if (lo >= hi) return;
  uint16_t* dst = (which ? a.v : a.k) + (s.row0 - s.past) * (a.c.kv * D) + head * D;
  const int64_t pitch = static_cast<int64_t>(a.c.kv) * D;
  const int64_t page = block < len / kBlock ? a.c.page(seq, block) : -1;
  const bool open = block == len / kBlock;  // the tail's tokens, up to len
  const uint16_t* tail = a.c.tail + ((static_cast<int64_t>(seq) * 2 + which) * a.c.kv + head) * (kBlock * D);
  if (page >= 0) {
    const int64_t place = (page * 2 + which) * a.c.kv + head;
    const float scale = a.c.scales[place];
    const u32x4* src = reinterpret_cast<const u32x4*>(a.c.codes + place * (kBlock * D));
    for (int i = tid; i < kBlock * D / 16; i += kThreads) {
      const int row = i & 15, g = (i >> 4) & 3, outer = i >> 6;
      const u32x4 w = src[i];
      constexpr int kC = D / 64;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
#pragma unroll
        for (int b = 0; b < 4; ++b) {
          // the byte selector is an immediate
          const float x = b == 0   ? __builtin_amdgcn_cvt_f32_fp8(w[e], 0)
                          : b == 1 ? __builtin_amdgcn_cvt_f32_fp8(w[e], 1)
                          : b == 2 ? __builtin_amdgcn_cvt_f32_fp8(w[e], 2)
                                   : __builtin_amdgcn_cvt_f32_fp8(w[e], 3);
          const int t = which ? e * 16 + g * 4 + b : (outer / kC) * 16 + row;
          const int d = which ? outer * 16 + row : (outer % kC) * 64 + g * 16 + 4 * e + b;
          tile[t][d] = held<T>(x, scale);
        }
      }
    }
  } else {
    for (int i = tid; i < kBlock * D; i += kThreads) {
      // the keys' tail is in the order of the tile, the values' is transposed
      const int t = which ? i % kBlock : i / D, d = which ? i / kBlock : i % D;
      tile[t][d] = open && block * kBlock + t < len ? tail[i] : 0;
    }
  }
  __syncthreads();
  for (int i = tid; i < (hi - lo) * kPer; i += kThreads) {
    const int at = lo + i / kPer, d = (i % kPer) * 8;
    const uint32_t* x = reinterpret_cast<const uint32_t*>(&tile[at - block * kBlock][d]);
    *reinterpret_cast<u32x4*>(dst + at * pitch + d) = u32x4{x[0], x[1], x[2], x[3]};
  }
}

// ------------------------------------------------------------------------------------------------
// Attention
// ------------------------------------------------------------------------------------------------

struct AttnArgs {
  Cache c;
  const uint16_t* q;
  int64_t q_tok, q_head;
  int64_t n_rows;
  int n_q, group;
  const int32_t* bounds;
  const int32_t* past;
  int max_new, max_len;
  float scale_log2;
  int window, sinks;  // window 0: every key
  int tiles, splits, per;  // tiles of rows per sequence and KV head; parts of the pages, pages of a part
  uint16_t* out;      // [n_rows, n_q, D]
  float* part_o;      // [n_rows, n_q, splits, D]
  float2* part_ml;    // [n_rows, n_q, splits]: maximum, sum
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

// Over the four lanes of one query column, 16 apart.
__device__ __forceinline__ float rows_max(float x) {
  const uint32_t u = __builtin_bit_cast(uint32_t, x);
  const auto r = __builtin_amdgcn_permlane16_swap(u, u, false, false);
  x = fmaxf(__builtin_bit_cast(float, static_cast<uint32_t>(r[0])), __builtin_bit_cast(float, static_cast<uint32_t>(r[1])));
  const uint32_t w = __builtin_bit_cast(uint32_t, x);
  const auto q = __builtin_amdgcn_permlane32_swap(w, w, false, false);
  return fmaxf(__builtin_bit_cast(float, static_cast<uint32_t>(q[0])), __builtin_bit_cast(float, static_cast<uint32_t>(q[1])));
}
__device__ __forceinline__ float rows_sum(float x) {
  x += __shfl_xor(x, 16, kWave);
  return x + __shfl_xor(x, 32, kWave);
}

// The 16 scores of a lane (tokens first + 16 t + 4 g + r) become weights exp2(c s - m) of a running
// maximum m; returns what the sums so far are multiplied by. kMask: tokens that the row does not see.
struct Softmax {
  float m = -__builtin_inff(), l = 0.f;
  __device__ __forceinline__ float step(f32x4 (&st)[4], float c, bool mask, int first, int g, int place, int window,
                                        int sinks) {
    if (mask) {
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int key = first + t * 16 + g * 4 + r;
          const bool seen = key <= place && (window == 0 || place - key < window || key < sinks);
          st[t][r] = seen ? st[t][r] : -__builtin_inff();
        }
    }
    float top = st[0][0];
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int r = 0; r < 4; ++r) top = fmaxf(top, st[t][r]);
    const float m_new = fmaxf(m, rows_max(top) * c);
    // a row that has seen no key yet keeps -inf, its weights are exp2(-inf - 0) = 0
    const float ref = m_new == -__builtin_inff() ? 0.f : m_new;
    const float alpha = __builtin_amdgcn_exp2f(m - ref);
    m = m_new;
    float sum = 0.f;
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        st[t][r] = __builtin_amdgcn_exp2f(__builtin_fmaf(st[t][r], c, -ref));
        sum += st[t][r];
      }
    l = l * alpha + sum;
    return alpha;
  }
};

// A workgroup: 16 (token, head) rows of one sequence and KV head against one part of its pages, a
// page per wavefront at a time, each with its own running maximum and sum; joined through LDS.
template <class T, int D>
__global__ __launch_bounds__(kThreads, 3) void cache_attn_kernel(AttnArgs a) {
  constexpr int kC = D / 64, kN = D / 16, kPitch = D + 4;
  __shared__ float part[kWaves][16][kPitch];
  __shared__ float stat[2][kWaves][16];
  const int tid = threadIdx.x, lane = tid & 63, col = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid / kWave);
  const int split = static_cast<int>(blockIdx.x % a.splits);
  int rest = static_cast<int>(blockIdx.x / a.splits);
  const int tile = rest % a.tiles;
  rest /= a.tiles;
  const int head = rest % a.c.kv, seq = rest / a.c.kv;
  const Span s = span_of(a.bounds, a.past, seq, a.n_rows, a.max_new, a.max_len);
  const int rows = s.n * a.group, r0 = tile * 16;
  if (r0 >= rows) return;
  const int len = s.past + s.n;
  const int row = min(r0 + col, rows - 1);  // the columns behind the last row repeat it
  const int at = row / a.group, place = s.past + at;
  const int lo_place = s.past + r0 / a.group, hi_place = s.past + min(r0 + 15, rows - 1) / a.group;
  const Visits visits(lo_place, hi_place, a.window, a.sinks);
  const int begin = split * a.per, end = min(visits.count, begin + a.per);
  if (begin >= end) return;
  const int qh = head * a.group + row % a.group;
  // the last visit is the open block, whose tokens are in the tail, where the rows reach it
  const bool open = hi_place / kBlock == len / kBlock;
  const int code_end = a.c.n_pages > 0 ? min(end, visits.count - (open ? 1 : 0)) : begin;

  half8 q[kC][2];
  {
    const uint16_t* p = a.q + (s.row0 + at) * a.q_tok + qh * a.q_head + g * 16;
#pragma unroll
    for (int c = 0; c < kC; ++c)
#pragma unroll
      for (int h = 0; h < 2; ++h) q[c][h] = *reinterpret_cast<const half8*>(p + c * 64 + h * 8);
  }
  f32x4 acc[kN];
#pragma unroll
  for (int n = 0; n < kN; ++n) acc[n] = f32x4{0.f, 0.f, 0.f, 0.f};
  Softmax soft;
  u32x4 kw[4 * kC], vw[kN];
  auto load_k = [&](int page) {
    const u32x4* src = reinterpret_cast<const u32x4*>(
                           a.c.codes + (static_cast<int64_t>(page) * 2 * a.c.kv + head) * (kBlock * D)) + lane;
#pragma unroll
    for (int t = 0; t < 4 * kC; ++t) kw[t] = __builtin_nontemporal_load(src + t * kWave);
  };
  auto load_v = [&](int page) {
    const u32x4* src = reinterpret_cast<const u32x4*>(
                           a.c.codes + ((static_cast<int64_t>(page) * 2 + 1) * a.c.kv + head) * (kBlock * D)) + lane;
#pragma unroll
    for (int n = 0; n < kN; ++n) vw[n] = __builtin_nontemporal_load(src + n * kWave);
  };

  // 64 of the wavefront's pages at a time: lane l holds the l-th one's place and scales
  for (int base = begin + wave; base < code_end; base += kWaves * kWave) {
    const int mine = base + kWaves * lane;
    int page_l = -1;
    float ks_l = 1.f, vs_l = 1.f;
    if (mine < code_end) {
      page_l = static_cast<int>(a.c.page(seq, visits.page(mine)));
      if (page_l >= 0) {
        ks_l = a.c.scales[static_cast<int64_t>(page_l) * 2 * a.c.kv + head];
        vs_l = a.c.scales[(static_cast<int64_t>(page_l) * 2 + 1) * a.c.kv + head];
      }
    }
    const int count = min((code_end - base + kWaves - 1) / kWaves, kWave);
    // what is no page is read as the pool's first one and seen by no row
    int page = __builtin_amdgcn_readlane(page_l, 0);
    load_k(max(page, 0));
    load_v(max(page, 0));
    auto step = [&](int i, auto more) {
      const float k_scale = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, ks_l), i));
      const float v_scale = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, vs_l), i));
      const int next = decltype(more)::value ? __builtin_amdgcn_readlane(page_l, i + 1) : 0;
      f32x4 st[4];
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        st[t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int c = 0; c < kC; ++c) {
          const u32x4 w = kw[t * kC + c];
          st[t] = T::mfma(T::codes(u32x2{w.x, w.y}), q[c][0], st[t]);
          st[t] = T::mfma(T::codes(u32x2{w.z, w.w}), q[c][1], st[t]);
        }
      }
      // the next page's keys are on their way while this one's weights and values are worked on, its
      // values during the next one's scores (the last page is a copy of its own without them: a
      // condition here would make every wait one for all loads)
      __builtin_amdgcn_sched_barrier(0);
      if constexpr (decltype(more)::value) load_k(max(next, 0));
      __builtin_amdgcn_sched_barrier(0);
      const int first = visits.page(base + kWaves * i) * kBlock;
      const bool all = page >= 0 && first + kBlock - 1 <= lo_place &&
                       (a.window == 0 || hi_place - first < a.window || first + kBlock <= a.sinks);
      const float alpha = soft.step(st, a.scale_log2 * k_scale, !all, page >= 0 ? first : 0x7fff0000, g, place,
                                    a.window, a.sinks);
      // P in fp16 whatever the operands' type: the values' codes are exact in it. The error is that of
      // a rounding to 11 bits, below the output's own.
      half8 p[2];
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          p[u][r] = static_cast<_Float16>(st[2 * u][r]);
          p[u][4 + r] = static_cast<_Float16>(st[2 * u + 1][r]);
        }
      if (page < 0) {
#pragma unroll
        for (int n = 0; n < kN; ++n) vw[n] = u32x4{0, 0, 0, 0};
      }
#pragma unroll
      for (int n = 0; n < kN; ++n) {
        f32x4 o = {0.f, 0.f, 0.f, 0.f};
        o = F16::mfma(F16::codes(u32x2{vw[n].x, vw[n].y}), p[0], o);
        o = F16::mfma(F16::codes(u32x2{vw[n].z, vw[n].w}), p[1], o);
        // the scale of the page's values in fp32: it may be past what fp16 holds
#pragma unroll
        for (int r = 0; r < 4; ++r) acc[n][r] = __builtin_fmaf(o[r], v_scale, acc[n][r] * alpha);
      }
      __builtin_amdgcn_sched_barrier(0);
      if constexpr (decltype(more)::value) load_v(max(next, 0));
      __builtin_amdgcn_sched_barrier(0);
      page = next;
    };
    for (int i = 0; i < count - 1; ++i) step(i, std::true_type{});
    step(count - 1, std::false_type{});
  }

  // the tail, by the wavefront whose turn it is
  if (open && visits.count - 1 >= begin && visits.count - 1 < end && (visits.count - 1 - begin) % kWaves == wave) {
    const uint16_t* tk = a.c.tail + (static_cast<int64_t>(seq) * 2 * a.c.kv + head) * (kBlock * D);
    const uint16_t* tv = tk + static_cast<int64_t>(a.c.kv) * (kBlock * D);
    const int first = len / kBlock * kBlock, left = len - first;
    f32x4 st[4];
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      st[t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int c = 0; c < kC; ++c)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const half8 w = *reinterpret_cast<const half8*>(tk + (t * 16 + col) * D + c * 64 + g * 16 + h * 8);
          st[t] = T::mfma(w, q[c][h], st[t]);
        }
    }
    const float alpha = soft.step(st, a.scale_log2, true, first, g, place, a.window, a.sinks);
    // the weights in the tail's type; for bfloat16 as two parts, so that they keep 16 bits
    half8 hi[2], lo[2];
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float x = st[2 * u + e / 4][e % 4];
        const uint16_t b = T::down(x);
        hi[u][e] = __builtin_bit_cast(_Float16, b);
        lo[u][e] = __builtin_bit_cast(_Float16, T::down(x - T::up(b)));
      }
#pragma unroll
    for (int n = 0; n < kN; ++n) {
#pragma unroll
      for (int r = 0; r < 4; ++r) acc[n][r] *= alpha;
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        uint64_t w[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          // what lies behind the sequence's tokens is no value
          const int t = (2 * u + e) * 16 + g * 4, there = min(max(left - t, 0), 4);
          w[e] = *reinterpret_cast<const uint64_t*>(tv + (n * 16 + col) * kBlock + t);
          w[e] &= there == 4 ? ~uint64_t{0} : (uint64_t{1} << (16 * there)) - 1;
        }
        struct Two { uint64_t x, y; };
        const half8 v = __builtin_bit_cast(half8, Two{w[0], w[1]});
        acc[n] = T::mfma(v, hi[u], acc[n]);
        if constexpr (__is_same(T, BF16)) acc[n] = T::mfma(v, lo[u], acc[n]);
      }
    }
  }

  float m = soft.m, l = soft.l;
  l = rows_sum(l);
  if (g == 0) {
    stat[0][wave][col] = m;
    stat[1][wave][col] = l;
  }
  __syncthreads();
  float top = stat[0][0][col];
#pragma unroll
  for (int w = 1; w < kWaves; ++w) top = fmaxf(top, stat[0][w][col]);
  const float mine = m == -__builtin_inff() ? 0.f : __builtin_amdgcn_exp2f(m - top);
#pragma unroll
  for (int n = 0; n < kN; ++n)
    *reinterpret_cast<f32x4*>(&part[wave][col][n * 16 + g * 4]) =
        f32x4{acc[n][0] * mine, acc[n][1] * mine, acc[n][2] * mine, acc[n][3] * mine};
  __syncthreads();
  const bool only = visits.count <= a.per;
  for (int i = tid; i < 16 * D / 4; i += kThreads) {
    const int c = i / (D / 4), d = (i % (D / 4)) * 4, r = r0 + c;
    if (r >= rows) break;
    float best = stat[0][0][c], sum = 0.f;
#pragma unroll
    for (int w = 1; w < kWaves; ++w) best = fmaxf(best, stat[0][w][c]);
    f32x4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      const float x = stat[0][w][c];
      sum += x == -__builtin_inff() ? 0.f : stat[1][w][c] * __builtin_amdgcn_exp2f(x - best);
      const f32x4 y = *reinterpret_cast<const f32x4*>(&part[w][c][d]);
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] += y[e];
    }
    const int64_t to = (s.row0 + r / a.group) * a.n_q + head * a.group + r % a.group;
    if (only) {
      const float inv = sum > 0.f ? 1.f / sum : sum == 0.f ? 0.f : sum;  // a sum that is NaN stays one
      u32x2 w;
      w.x = T::down(o[0] * inv) | static_cast<uint32_t>(T::down(o[1] * inv)) << 16;
      w.y = T::down(o[2] * inv) | static_cast<uint32_t>(T::down(o[3] * inv)) << 16;
      *reinterpret_cast<u32x2*>(a.out + to * D + d) = w;
    } else {
      *reinterpret_cast<f32x4*>(a.part_o + (to * a.splits + split) * D + d) = o;
      if (d == 0) a.part_ml[to * a.splits + split] = make_float2(best, sum);
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

// The parts of one row and head, joined in their order: 4 kLanes columns a workgroup, its groups of
// kLanes threads take every so many-th part, all loads on their way before the weights are known.
template <class T, int D, int kLanes>
__global__ __launch_bounds__(kThreads) void cache_join_kernel(AttnArgs a) {
  constexpr int kGroups = kThreads / kLanes, kEach = 8, kSlices = D / (4 * kLanes);
  __shared__ float weight[kSplits];
  __shared__ f32x4 sums[kGroups][kLanes];
  const int tid = threadIdx.x, lane = tid & 63;
  const int slice = static_cast<int>(blockIdx.x % kSlices);
  int rest = static_cast<int>(blockIdx.x / kSlices);
  const int qh = rest % a.n_q;
  rest /= a.n_q;
  const int at = rest % a.max_new, seq = rest / a.max_new;
  const Span s = span_of(a.bounds, a.past, seq, a.n_rows, a.max_new, a.max_len);
  if (at >= s.n) return;
  const int rows = s.n * a.group, r0 = (at * a.group + qh % a.group) / 16 * 16;
  const Visits visits(s.past + r0 / a.group, s.past + min(r0 + 15, rows - 1) / a.group, a.window, a.sinks);
  const int parts = (visits.count + a.per - 1) / a.per;
  if (parts <= 1) return;  // written by its one part
  const int64_t to = (s.row0 + at) * a.n_q + qh;
  const int grp = tid / kLanes, d = slice * 4 * kLanes + (tid % kLanes) * 4;
  const float* p = a.part_o + to * a.splits * D + d;
  f32x4 o[kEach];
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    const int j = grp + i * kGroups;
    o[i] = j < parts ? *reinterpret_cast<const f32x4*>(p + static_cast<int64_t>(j) * D) : f32x4{0.f, 0.f, 0.f, 0.f};
  }
  // every wavefront takes all weights
  constexpr int kPer = kSplits / kWave;
  float2 ml[kPer];
  float top = -__builtin_inff();
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int j = lane + i * kWave;
    ml[i] = j < parts ? a.part_ml[to * a.splits + j] : make_float2(-__builtin_inff(), 0.f);
    top = fmaxf(top, ml[i].x);
  }
  top = lanes_max(top);
  float sum = 0.f;
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const float w = ml[i].x == -__builtin_inff() ? 0.f : __builtin_amdgcn_exp2f(ml[i].x - top);
    sum += ml[i].y * w;
    if (tid < kWave) weight[lane + i * kWave] = w;
  }
  sum = lanes_sum(sum);
  __syncthreads();
  f32x4 total = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    const int j = grp + i * kGroups;
    if (j < parts) {
#pragma unroll
      for (int e = 0; e < 4; ++e) total[e] += weight[j] * o[i][e];
    }
  }
  sums[grp][tid % kLanes] = total;
  __syncthreads();
  if (grp != 0) return;
  const int used = min(kGroups, parts);
  for (int i = 1; i < used; ++i) {
    const f32x4 x = sums[i][tid];
#pragma unroll
    for (int e = 0; e < 4; ++e) total[e] += x[e];
  }
  const float inv = sum > 0.f ? 1.f / sum : sum == 0.f ? 0.f : sum;
  u32x2 w;
  w.x = T::down(total[0] * inv) | static_cast<uint32_t>(T::down(total[1] * inv)) << 16;
  w.y = T::down(total[2] * inv) | static_cast<uint32_t>(T::down(total[3] * inv)) << 16;
  *reinterpret_cast<u32x2*>(a.out + to * D + d) = w;
}

constexpr int kPerCu = 3;  // workgroups of the attention that a CU holds

// How an attention call splits its pages: enough workgroups to fill every CU, parts of at least a page
// per wavefront.
struct Plan {
  int64_t tiles, splits, per;
};
Plan plan_of(int64_t n_seqs, int64_t kv, int64_t group, int64_t max_new, int64_t max_len, int64_t window,
             int64_t sinks) {
  Plan p;
  sinks = std::min(sinks, max_len);
  p.tiles = (max_new * group + 15) / 16;
  int64_t visits = (max_len + kBlock - 1) / kBlock;
  if (window > 0) visits = std::min(visits, (window + 15 + 63) / kBlock + 1 + (sinks + kBlock - 1) / kBlock);
  const int64_t base = n_seqs * kv * p.tiles;
  const int64_t want = std::max<int64_t>(1, std::min<int64_t>(kSplits, kPerCu * device_cus() / std::max<int64_t>(base, 1)));
  p.per = std::max<int64_t>((visits + want - 1) / want, kWaves);
  p.splits = std::max<int64_t>((visits + p.per - 1) / p.per, 1);
  return p;
}

bool cache_shape(int32_t n_kv, int32_t head_dim, int32_t dtype, int32_t n_seqs, int64_t n_pages, int32_t width,
                 int64_t n_rows) {
  return n_kv >= 1 && n_kv <= 1024 && (head_dim == 64 || head_dim == 128) &&
         (dtype == TALM_F16 || dtype == TALM_BF16) && n_seqs >= 0 && n_pages >= 0 && n_pages < (int64_t{1} << 31) &&
         width >= 0 && width <= (1 << 24) && n_rows >= 0 && n_rows < (int64_t{1} << 31);
}

bool strides_fit(int64_t tok, int64_t head) { return tok % 8 == 0 && head % 8 == 0 && tok >= 0 && head >= 0; }

}  // namespace
}  // namespace talm

using namespace talm;

#define TALM_CACHE_KERNEL(name, grid, args)                                                                   \
  do {                                                                                                        \
    const dim3 g_(static_cast<unsigned>(grid)), b_(kThreads);                                                 \
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
              q_stride_tok, q_stride_head, n_q_heads, q_out, 0};
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
  TALM_CACHE_KERNEL(LAUNCH, a.kv_items + turns, a);
#undef LAUNCH
  return check_launch("cache_write");
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
  const ReadArgs a{Cache{codes, scales, tail, table, n_pages, width, n_seqs, n_kv_heads}, length, bounds, past, n_rows,
                   max_new, width * kBlock, (max_new + kBlock - 1) / kBlock + 1, k, v};
  const int64_t items = static_cast<int64_t>(n_seqs) * n_kv_heads * 2 * a.chunks;
  if (items > 0x7fffffff) return fail(TALM_EINVAL, "cache_read: too many tokens");
  const hipStream_t st = as_stream(stream);
#define LAUNCH(T, D, grid, block, args) hipLaunchKernelGGL((cache_read_kernel<T, D>), grid, block, 0, st, args)
  TALM_CACHE_KERNEL(LAUNCH, items, a);
#undef LAUNCH
  return check_launch("cache_read");
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
  const Plan p = plan_of(n_seqs, n_kv_heads, n_q_heads / n_kv_heads, max_new, max_len, window, sinks);
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
  const Plan p = plan_of(n_seqs, n_kv_heads, n_q_heads / n_kv_heads, max_new, max_len, window, sinks);
  float* part_o = static_cast<float*>(workspace);
  AttnArgs a{Cache{codes, scales, tail, table, n_pages, width, n_seqs, n_kv_heads}, q, q_stride_tok, q_stride_head,
             n_rows, n_q_heads, n_q_heads / n_kv_heads, bounds, past, max_new, std::min(max_len, width * kBlock),
             scale * 1.44269504088896340736f, window, std::min(sinks, max_len), static_cast<int>(p.tiles), static_cast<int>(p.splits),
             static_cast<int>(p.per), out, part_o,
             reinterpret_cast<float2*>(part_o ? part_o + n_rows * n_q_heads * p.splits * head_dim : nullptr)};
  const int64_t items = static_cast<int64_t>(n_seqs) * n_kv_heads * p.tiles * p.splits;
  const int64_t joins = p.splits > 1 ? static_cast<int64_t>(n_seqs) * max_new * n_q_heads : 0;
  if (items > 0x7fffffff || joins * (head_dim / 32) > 0x7fffffff) return fail(TALM_EINVAL, "cache_attn: too many rows");
  const hipStream_t st = as_stream(stream);
#define LAUNCH(T, D, grid, block, args) hipLaunchKernelGGL((cache_attn_kernel<T, D>), grid, block, 0, st, args)
  TALM_CACHE_KERNEL(LAUNCH, items, a);
#undef LAUNCH
  if (const int status = check_launch("cache_attn")) return status;
  if (joins == 0) return TALM_OK;
  // a whole head's columns a workgroup where its groups reach the parts in eight steps, else 32
  const bool few = p.splits <= 8 * (kThreads / (head_dim / 4));
  const int64_t slices = few ? 1 : head_dim / 32;
#define LAUNCH(T, D, grid, block, args)                                                  \
  do {                                                                                   \
    if (few)                                                                             \
      hipLaunchKernelGGL((cache_join_kernel<T, D, D / 4>), grid, block, 0, st, args);    \
    else                                                                                 \
      hipLaunchKernelGGL((cache_join_kernel<T, D, 8>), grid, block, 0, st, args);        \
  } while (0)
  TALM_CACHE_KERNEL(LAUNCH, joins * slices, a);
#undef LAUNCH
  return check_launch("cache_attn");
}
