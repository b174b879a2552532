// Products of a few tokens (1 .. 32) with a weight W [rows, cols] held in the layer group's NF4 form,
// for the calls that answer token by token: out = x W^T + bias (+ LoRA adapters, ts B^T). Every weight is
// read once as its 4-bit code, with its block's absmax code and second-level scale, and never written out;
// the fp16 weights are bit-identical to talm_nf4_group_dequant's (solution/qgroup.py:72-99), the products fp32.
//
// The weights are the A operand of v_mfma_f32_16x16x32_f16, the tokens the B operand. A lane takes
// whole 64-weight blocks (32 contiguous bytes of codes, one scale); the reduction's order is free, so
// eight MFMAs take a block's eight-weight words as they lie, against the same columns of x. Sixteen
// operand rows are R = 16 / P rows of W times P parts of the reduction (a unit: 256 P columns); the
// operand's columns are the tokens times the same P parts, and the blocks of the result where both
// parts agree are summed: few tokens leave operand columns free, and small tiles give a W of few
// rows enough workgroups. The wavefronts of a workgroup split the units, joined through LDS in order.
//
// Two ways to look a code up, by the size of W:
//   rows kernel  a table of the block's 16 scaled levels in the lane's registers (nf4_code.h), 310 VALU
//                instructions per block, half of them byte permutes;
//   lut kernel   per byte of codes its two levels from a table in LDS (one ds_read_b64 through an
//                address made by one byte permute), scaled and packed: 140 instructions per block.
//                The table stands in 32 copies, lane l reading copy l % 32, so that the 32 lanes of a
//                read phase meet 32 different bank pairs whatever their codes are; its 64 KiB cost 1 us
//                to fill and make one workgroup per CU, whose wavefronts walk all of its tiles, joined as
//                many at a time as the LDS has room for.
// A lane's share of x is 16 bytes of 64 columns from the next lane group's: loaded straight, a load
// instruction of many tokens touches 64 cache lines, and the eight that share them run behind each other
// through a smaller cache. With many tokens x comes in pieces of 64 bytes and changes places in LDS
// (us, straight / through LDS: W [17920, 1536] 16 tokens 9.7 / 8.3, 32 tokens 13.5 / 10.1; [1536, 8960] 16
// tokens 14.3 / 10.1, 32 tokens 21.8 / 13.3; several units per wavefront, [3584, 18944]: 2 tokens 16.9 / 18.5,
// 4 20.4 / 18.6, 8 27.7 / 20.0; [1536, 8960] 5 tokens 7.7 / 8.0, 6 8.3 / 8.0).
// MI355X, us, rows / lut: W [2048, 1536] 1 token 3.1 / 5.6, 32 tokens 6.0 / 6.1; [8960, 1536] 7.2 / 6.0,
// 14.3 / 8.6; lut: [17920, 1536] 7.1 and 10.1 (2.0 TB/s of codes and scales), [1536, 8960] 6.8 and 13.3,
// [152064, 1536] 28 and 42 (4.3 TB/s, 2.9). What bounds one token: a launch (1.2 us), one memory
// round trip with the whole of W in flight, the lookups behind it (LDS and VALU 1.4 us each) and the
// join, one after the other; many tokens: x's way through L2 and LDS, and the lookups.
// These read one W again and again, which then lies in the L2. With the W of 28 layers in turn (45, 33, 400 and 200 MB:
// from the last-level cache, gate|up's from memory), one token / 32: q|k|v [2048, 1536] 4.0 / 6.9 us, o 3.6 / 6.5,
// gate|up 8.0 / 11.5, down 6.8 / 13.2; all of a model's products behind each other, 650 MB from memory, 23.6 / 40.7 a
// layer, eight tokens 26.9. An adapter's sum in the store adds 0.1 to
// 0.6 us (1.2 at gate|up of 32 tokens); its down product is a launch in front: q|k|v with q's and v's adapters 8.3
// and 13.0 us, 9.3 and 14.0 over 28 layers.
// Not kept: three tiles' weights ahead in registers (1 token, [17920, 1536] 8.4 us, [2048, 8192] 7.6 for 6.3); the
// rows kernel's lookups as a loop (3.3 us for 3.15).
#include "mfma_tile.h"
#include "nf4_code.h"

#include <algorithm>

namespace talm {
namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));

struct GemvArgs {
  const uint16_t* x;  // [M][ldx]
  int64_t ldx;
  int M, rows, cols;
  const uint8_t* packed;
  const uint8_t* absmax8;
  const float* code;
  const float* absmax2;
  const float* offset2;
  int shift2;            // log2 of the blocks per second-level scale
  const uint16_t* bias;  // [rows] or null
  const uint16_t* ts;    // [M][ldt]: the scaled down products of up to two LoRA adapters of rank 16, or null
  int64_t ldt;
  const uint16_t* b[2];  // [hi - lo][16]: adapter g adds ts_g b_g^T to rows lo .. hi - 1
  int lo[2], hi[2];
  uint16_t* out;         // [M][ldo]
  int64_t ldo;
  int units;
  int tiles_per_wg, round, unit_waves, groups;  // the lut kernel: wavefront w takes units w % unit_waves, .. of
                                         // tiles w / unit_waves, .. of the workgroup's
};

constexpr int kGemvMaxWaves = 16;
constexpr int kGemvTokens = 32;

// A unit's weights of one lane, as loaded: a block's codes and its scale's inputs.
struct GemvBlock {
  uint4 lo, hi;
  uint8_t a8;
  float s2, o2;
};

// LDS operations of a wavefront complete in order: its lanes see each other's once the compiler keeps theirs.
__device__ __forceinline__ void wave_sync() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

constexpr int kStageBytes = 4096;

// A lane's place in its operands, and its loads of W from the workgroup's first row on and of x.
template <int P, int TB>
struct GemvLane {
  static constexpr int R = 16 / P;  // rows of W per tile, and tokens per block
  int row0, wr, part, g;            // wr: the lane's row of a tile (A) and token of a block (B)
  int64_t first;                    // the workgroup's first weight (those after it fit 31 bits)
  __amdgpu_buffer_rsrc_t rw, rs, rx;
  __device__ __forceinline__ GemvLane(const GemvArgs& a, int row, int lane)
      : row0(row), wr(lane & (R - 1)), part((lane & 15) / R), g(lane >> 4),
        first(static_cast<int64_t>(row) * a.cols) {
    rw = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(a.packed + first / 2), 0, 0x7fffffff, 0x00020000);
    rs = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(a.absmax8 + first / 64), 0, 0x7fffffff, 0x00020000);
    rx = buffer_rsrc(a.x);
  }
  __device__ __forceinline__ int column(int unit) const { return (unit * P + part) * 256 + 64 * g; }
  // A lane outside W reads codes and scales of 0, against columns of x that read 0, or for rows that
  // are not stored.
  __device__ __forceinline__ void load_w(const GemvArgs& a, int tile, int unit, GemvBlock& w) const {
    const int k = column(unit), row = R * tile + wr;
    const bool in = k < a.cols && row0 + row < a.rows;
    const uint32_t e = static_cast<uint32_t>(row * a.cols + k);
    w.lo = __builtin_bit_cast(uint4, __builtin_amdgcn_raw_buffer_load_b128(rw, in ? e / 2 : kOob, 0, 0));
    w.hi = __builtin_bit_cast(uint4, __builtin_amdgcn_raw_buffer_load_b128(rw, in ? e / 2 + 16 : kOob, 0, 0));
    w.a8 = __builtin_amdgcn_raw_buffer_load_b8(rs, in ? e / 64 : kOob, 0, 0);
    const int64_t group = in ? ((first + e) >> 6) >> a.shift2 : 0;
    w.s2 = in ? a.absmax2[group] : 0.f;
    w.o2 = in ? a.offset2[group] : 0.f;
  }
  __device__ __forceinline__ void load_x(const GemvArgs& a, int unit, uint4 (&x)[TB][8]) const {
    const int k = column(unit);
#pragma unroll
    for (int b = 0; b < TB; ++b) {
      const int tok = wr + R * b;
      const uint32_t off = k < a.cols && tok < a.M ? static_cast<uint32_t>((tok * a.ldx + k) * 2) : kOob;
#pragma unroll
      for (int j = 0; j < 8; ++j)
        x[b][j] = __builtin_bit_cast(uint4, __builtin_amdgcn_raw_buffer_load_b128(rx, off, 16 * j, 0));
    }
  }
  // The same operand, its global loads in pieces of 64 bytes: half `p` of a token's four blocks by 16
  // lanes, four tokens at a time, then through the wavefront's kStageBytes of LDS, 16 tokens' halves at a
  // time. Chunk c (16 bytes) of token n lies at chunk c ^ n: the lanes of a read phase take 16 different.
  __device__ __forceinline__ void fetch_rows(const GemvArgs& a, int b, int unit, int lane, uint4 (&raw)[8]) const {
    const int c = lane & 15;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int n = 4 * (i & 3) + (lane >> 4), tok = R * b + (n & (R - 1));
      const int k = (unit * P + n / R) * 256 + 64 * (c >> 2) + 8 * (c & 3);
      const uint32_t off = k < a.cols && tok < a.M ? static_cast<uint32_t>((tok * a.ldx + k) * 2) : kOob;
      raw[i] = __builtin_bit_cast(uint4, __builtin_amdgcn_raw_buffer_load_b128(rx, off, 64 * (i >> 2), 0));
    }
  }
  __device__ __forceinline__ void stage_half(unsigned char* slice, int lane, const uint4* raw, uint4* x) const {
    const int n = lane & 15;
    wave_sync();  // the reads of the half before
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int row = 4 * i + (lane >> 4);
      *reinterpret_cast<uint4*>(slice + row * 256 + ((n ^ row) << 4)) = raw[i];
    }
    wave_sync();
#pragma unroll
    for (int j = 0; j < 4; ++j) x[j] = *reinterpret_cast<const uint4*>(slice + n * 256 + (((4 * g + j) ^ n) << 4));
  }
  // The lane's accumulators to its wavefront's slot: element v is operand row 4 (lane / 16) + v.
  __device__ __forceinline__ void leave(const f32x4 (&acc)[TB], float (&slot)[TB][P][R][R + 1]) const {
#pragma unroll
    for (int b = 0; b < TB; ++b)
#pragma unroll
      for (int v = 0; v < 4; ++v) {
        const int r = 4 * g + v;
        if (r / R == part) slot[b][part][r % R][wr] = acc[b][v];
      }
  }
};

// The sum of element (row, token) over `n` wavefronts' slots, in order; four slots' loads at a time.
template <int P, int R, class Slot>
__device__ __forceinline__ float gemv_join(const Slot* slot, int n, int b, int row, int token) {
  float sum = 0.f;
  for (int v0 = 0; v0 < n; v0 += 4) {
    float f[4][P];
#pragma unroll
    for (int v = 0; v < 4; ++v)
#pragma unroll
      for (int p = 0; p < P; ++p) f[v][p] = slot[min(v0 + v, n - 1)][b][p][row][token];
#pragma unroll
    for (int v = 0; v < 4; ++v)
#pragma unroll
      for (int p = 0; p < P; ++p) sum += v0 + v < n ? f[v][p] : 0.f;
  }
  return sum;
}

// The sum of the joined parts, bias and adapters, rounded and stored.
__device__ __forceinline__ void gemv_store(const GemvArgs& a, int row, int token, float sum) {
  if (a.bias) sum += h2f(a.bias[row]);
  if (a.ts) {
#pragma unroll
    for (int ad = 0; ad < 2; ++ad)
      if (row >= a.lo[ad] && row < a.hi[ad]) {
        const uint16_t* tp = a.ts + static_cast<int64_t>(token) * a.ldt + 16 * ad;
        const uint16_t* bp = a.b[ad] + static_cast<int64_t>(row - a.lo[ad]) * 16;
#pragma unroll
        for (int q = 0; q < 16; ++q) sum += h2f(tp[q]) * h2f(bp[q]);
      }
  }
  a.out[static_cast<int64_t>(token) * a.ldo + row] = f2h(sum);
}

// One workgroup per tile, a wavefront per unit (or several), the next unit's loads in flight.
template <int P, int TB>
__global__ __launch_bounds__(64 * kGemvMaxWaves) void nf4_gemv_rows_kernel(GemvArgs a) {
  constexpr int R = 16 / P;
  __shared__ float table[256];
  __shared__ float red[kGemvMaxWaves][TB][P][R][R + 1];
  const int tid = threadIdx.x, waves = blockDim.x >> 6;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int row0 = blockIdx.x * R;
  const GemvLane<P, TB> ln(a, row0, tid & 63);
  f32x4 acc[TB];
#pragma unroll
  for (int b = 0; b < TB; ++b) acc[b] = f32x4{0.f, 0.f, 0.f, 0.f};
  // the code table's load first: loads return in order, and its LDS write then waits for none of the
  // weights', whose first unit's fly meanwhile
  const float code = tid < 256 ? a.code[tid] : 0.f;
  GemvBlock w, next;
  constexpr bool kAhead = TB == 1;  // x too (two blocks of tokens would spill)
  uint4 x[TB][8], x_next[kAhead ? TB : 1][8];
  int u = wave;
  if (u < a.units) {
    ln.load_w(a, 0, u, w);
    ln.load_x(a, u, x);
  }
  if (tid < 256) table[tid] = code;
  for (int i = tid + blockDim.x; i < 256; i += blockDim.x) table[i] = a.code[i];
  lds_barrier();
  for (; u < a.units; u += waves) {
    const bool more = u + waves < a.units;
    if (more) {
      ln.load_w(a, 0, u + waves, next);
      if constexpr (kAhead) ln.load_x(a, u + waves, x_next);
    }
    const Nf4Table tab = nf4_table(block_scale(table[w.a8], w.s2, w.o2));
    const uint32_t words[8] = {w.lo.x, w.lo.y, w.lo.z, w.lo.w, w.hi.x, w.hi.y, w.hi.z, w.hi.w};
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const half8_t wf = __builtin_bit_cast(half8_t, nf4_lookup_word(words[j], tab));
#pragma unroll
      for (int b = 0; b < TB; ++b)
        acc[b] = __builtin_amdgcn_mfma_f32_16x16x32_f16(wf, __builtin_bit_cast(half8_t, x[b][j]), acc[b], 0, 0, 0);
    }
    if (more) {
      w = next;
      if constexpr (!kAhead) ln.load_x(a, u + waves, x);
#pragma unroll
      for (int b = 0; b < (kAhead ? TB : 0); ++b)
#pragma unroll
        for (int j = 0; j < 8; ++j) x[b][j] = x_next[b][j];
    }
  }
  ln.leave(acc, red[wave]);
  __syncthreads();
  for (int i = tid; i < TB * R * R; i += blockDim.x) {
    const int r = i % R, tok = i / R % R, b = i / (R * R);
    if (row0 + r >= a.rows || tok + R * b >= a.M) continue;
    gemv_store(a, row0 + r, tok + R * b, gemv_join<P, R>(red, waves, b, r, tok));
  }
}

constexpr int kLutBytes = 256 * 256;  // 256 bytes of codes x 32 copies of their two levels

// One workgroup per CU and a.tiles_per_wg tiles, joined a.round tiles at a time.
enum LutX {
  kEachUnit,   // a wavefront walks several units, and loads the x of each
  kOneUnit,    // it has one, whose x it keeps
  kOneStaged,  // the same, x loaded through LDS, where the results go later
  kEachStaged  // several, the x of each through LDS, half by half where the products take it
};
template <LutX kX>
struct LutRoom {  // wavefronts, and LDS: 160 KiB or less of the lookup table, absmax's, the x slices and
                  // the wavefronts' results of a round of tiles
  static constexpr int kWaves = kX == kEachStaged ? 12 : kGemvMaxWaves;
  static constexpr int kSlices = kX == kEachStaged ? kWaves * kStageBytes : 0;
  static constexpr int kRedFloats = kX == kEachStaged ? 11 * 1024 : 20 * 1024;
  static_assert(kX != kOneStaged || kWaves * kStageBytes <= kRedFloats * 4, "the slices lie in the results' room");
  static constexpr int kBytes = kLutBytes + 1024 + kSlices + kRedFloats * 4;
  static_assert(kBytes <= 160 * 1024, "LDS");
};
template <int P, int TB, LutX kX>
__global__ __launch_bounds__(64 * LutRoom<kX>::kWaves) void nf4_gemv_lut_kernel(GemvArgs a) {
  constexpr int R = 16 / P;
  __shared__ __attribute__((aligned(1024))) unsigned char smem[LutRoom<kX>::kBytes];
  float* table = reinterpret_cast<float*>(smem + kLutBytes);
  typedef float Slot[TB][P][R][R + 1];
  Slot* red = reinterpret_cast<Slot*>(smem + kLutBytes + 1024 + LutRoom<kX>::kSlices);  // [tile][unit wavefront]
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int uw = wave % a.unit_waves, grp = wave / a.unit_waves;
  const int row0 = blockIdx.x * a.tiles_per_wg * R;
  const int n_tiles = min(a.tiles_per_wg, (a.rows - row0 + R - 1) / R);
  const GemvLane<P, TB> ln(a, row0, lane);
  const float code = tid < 256 ? a.code[tid] : 0.f;  // first, as above
  unsigned char* slice = smem + kLutBytes + 1024 + wave * kStageBytes;
  GemvBlock w;
  uint4 x[kX == kEachStaged ? 1 : TB][8], raw[kX == kEachStaged ? TB : 1][8];
  int t = grp, u = uw;
  const bool any = t < n_tiles;
  auto fetch = [&](int unit) __attribute__((always_inline)) {
    if constexpr (kX == kEachStaged)
#pragma unroll
      for (int b = 0; b < TB; ++b) ln.fetch_rows(a, b, unit, lane, raw[b]);
  };
  if (any) {
    ln.load_w(a, t, u, w);
    if constexpr (kX == kOneStaged) ln.fetch_rows(a, 0, u, lane, raw[0]);
    else if constexpr (kX == kEachStaged) fetch(u);
    else ln.load_x(a, u, x);
  }
  // copy c of byte e's levels at e * 256 + 8 c: a thread writes two copies, a wavefront four bytes of
  // one high nibble (the levels through scalar loads: no wait for the weights either)
  for (int e0 = 4 * wave; e0 < 256; e0 += blockDim.x >> 4) {
    const float* l = kNF4Levels + (e0 & 15);
    const float hi = kNF4Levels[e0 >> 4], l0 = l[0], l1 = l[1], l2 = l[2], l3 = l[3];
    const float lo = lane < 32 ? (lane < 16 ? l0 : l1) : (lane < 48 ? l2 : l3);
    *reinterpret_cast<float4*>(smem + e0 * 256 + lane * 16) = make_float4(hi, lo, hi, lo);
  }
  if (tid < 256) table[tid] = code;
  for (int i = tid + blockDim.x; i < 256; i += blockDim.x) table[i] = a.code[i];
  if constexpr (kX == kOneStaged)
    if (any) {
#pragma unroll
      for (int b = 0; b < TB; ++b) {
        if (b) ln.fetch_rows(a, b, u, lane, raw[0]);  // not with the first 16 tokens': 32 registers would be spilled
        ln.stage_half(slice, lane, raw[0], x[b]);
        ln.stage_half(slice, lane, raw[0] + 4, x[b] + 4);
      }
    }
  lds_barrier();
  // The first step needs all of its loads anyway; without this wait the compiler, which sees a path that skipped
  // their uses, would wait for them inside the loop, and so for the next step's.
  if constexpr (kX != kEachUnit) __builtin_amdgcn_s_waitcnt(0x0f70);  // vmcnt(0)
  const uint32_t copy = (lane & 31) * 8;
  f32x4 acc[TB];
#pragma unroll
  for (int b = 0; b < TB; ++b) acc[b] = f32x4{0.f, 0.f, 0.f, 0.f};
  for (int first = 0; first < n_tiles; first += a.round) {
    const int end = min(n_tiles, first + a.round);
    while (t < end) {
      int tn = t, un = u + a.unit_waves;  // the next step: this tile's next unit, or the next tile
      if (un >= a.units) {
        un = uw;
        tn += a.groups;
      }
      const bool more = tn < n_tiles;
      GemvBlock next;
      if (more) ln.load_w(a, tn, un, next);
      const float scale = block_scale(table[w.a8], w.s2, w.o2);
      const uint32_t words[8] = {w.lo.x, w.lo.y, w.lo.z, w.lo.w, w.hi.x, w.hi.y, w.hi.z, w.hi.w};
      auto levels = [&](uint32_t word) __attribute__((always_inline)) {
        uint32_t h[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) {  // byte q of the word to bits 8..15, the copy below it
          const uint32_t at = __builtin_amdgcn_perm(word, copy, 0x0c0c0400u + (static_cast<uint32_t>(q) << 8));
          const float2 f = *reinterpret_cast<const float2*>(smem + at);
          const nf4_float2_t wq = {mul_f32(f.x, scale), mul_f32(f.y, scale)};
          h[q] = __builtin_bit_cast(uint32_t, __builtin_convertvector(wq, nf4_half2_t));
        }
        return __builtin_bit_cast(half8_t, make_uint4(h[0], h[1], h[2], h[3]));
      };
      if constexpr (kX == kEachStaged) {
#pragma unroll
        for (int p = 0; p < 2; ++p) {
          half8_t wf[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) wf[j] = levels(words[4 * p + j]);
#pragma unroll
          for (int b = 0; b < TB; ++b) {
            ln.stage_half(slice, lane, raw[b] + 4 * p, x[0]);
#pragma unroll
            for (int j = 0; j < 4; ++j)
              acc[b] = __builtin_amdgcn_mfma_f32_16x16x32_f16(wf[j], __builtin_bit_cast(half8_t, x[0][j]), acc[b], 0,
                                                              0, 0);
          }
        }
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const half8_t wf = levels(words[j]);
#pragma unroll
          for (int b = 0; b < TB; ++b)
            acc[b] = __builtin_amdgcn_mfma_f32_16x16x32_f16(wf, __builtin_bit_cast(half8_t, x[b][j]), acc[b], 0, 0, 0);
        }
      }
      if (tn != t) {  // the tile is done
        ln.leave(acc, red[(t - first) * a.unit_waves + uw]);
#pragma unroll
        for (int b = 0; b < TB; ++b) acc[b] = f32x4{0.f, 0.f, 0.f, 0.f};
      }
      t = tn;
      u = un;
      if (more) {
        w = next;
        if constexpr (kX == kEachStaged) fetch(u);
        else if constexpr (kX == kEachUnit) ln.load_x(a, u, x);
      }
    }
    lds_barrier();
    const int rows = (end - first) * R, row1 = row0 + first * R;
    for (int i = tid; i < rows * TB * R; i += blockDim.x) {
      const int rl = i % rows, token = i / rows, b = token / R;
      if (row1 + rl >= a.rows || token >= a.M) continue;
      const Slot* slot = red + rl / R * a.unit_waves;
      gemv_store(a, row1 + rl, token, gemv_join<P, R>(slot, a.unit_waves, b, rl % R, token % R));
    }
    if (end < n_tiles) lds_barrier();
  }
}

template <int P, int TB, LutX kX>
void launch_lut(GemvArgs a, hipStream_t s) {
  constexpr int R = 16 / P, most = LutRoom<kX>::kWaves;
  const int tiles = (a.rows + R - 1) / R, turns = (a.units + most - 1) / most;
  a.unit_waves = (a.units + turns - 1) / turns;
  const int room = LutRoom<kX>::kRedFloats / (a.unit_waves * TB * P * R * (R + 1));
  a.tiles_per_wg = std::min((tiles + device_cus() - 1) / device_cus(), 0x7fffffff / (R * a.cols));  // 32-bit offsets
  a.groups = std::max(1, std::min(std::min(a.tiles_per_wg, room), most / a.unit_waves));
  a.round = room / a.groups * a.groups;
  hipLaunchKernelGGL((nf4_gemv_lut_kernel<P, TB, kX>),
                     dim3(static_cast<unsigned>((tiles + a.tiles_per_wg - 1) / a.tiles_per_wg)),
                     dim3(64 * a.unit_waves * a.groups), 0, s, a);
}

template <int P, int TB>
void launch_rows(GemvArgs a, hipStream_t s) {
  constexpr int R = 16 / P;
  a.units = (a.cols + 256 * P - 1) / (256 * P);
  const int turns = (a.units + kGemvMaxWaves - 1) / kGemvMaxWaves, waves = (a.units + turns - 1) / turns;
  hipLaunchKernelGGL((nf4_gemv_rows_kernel<P, TB>), dim3(static_cast<unsigned>((a.rows + R - 1) / R)),
                     dim3(64 * waves), 0, s, a);
}

// The way of x: through LDS from 9 tokens on (which two parts hold as two blocks), from 6 on where a wavefront
// has several units (figures above).
template <int P, int TB>
void launch_lut_form(GemvArgs a, hipStream_t s) {
  a.units = (a.cols + 256 * P - 1) / (256 * P);
  const bool one = a.units <= kGemvMaxWaves;
  if constexpr (TB == 2) {
    if (one) launch_lut<P, TB, kOneStaged>(a, s);
    else launch_lut<P, TB, kEachStaged>(a, s);
  } else if (one) {
    if constexpr (P == 1)
      if (a.M > 8) return launch_lut<P, TB, kOneStaged>(a, s);
    launch_lut<P, TB, kOneUnit>(a, s);
  } else if (a.M > 5) {
    launch_lut<P, TB, kEachStaged>(a, s);
  } else {
    launch_lut<P, TB, kEachUnit>(a, s);
  }
}

}  // namespace
}  // namespace talm

using namespace talm;

TALM_API int talm_nf4_gemv(const uint16_t* x, int64_t ldx, int64_t n_tokens, const uint8_t* packed,
                           const uint8_t* absmax8, const float* code, const float* absmax2, const float* offset2,
                           int64_t rows, int64_t cols, int32_t qblock, int32_t qblock2, const uint16_t* bias,
                           const uint16_t* ts, int64_t ldt, const uint16_t* b0, int64_t lo0, int64_t hi0,
                           const uint16_t* b1, int64_t lo1, int64_t hi1, uint16_t* out, int64_t ldo,
                           void* stream) {
  if (qblock != 64 || qblock2 < 1 || (qblock2 & (qblock2 - 1)))
    return fail(TALM_EINVAL, "nf4_gemv: blocks of %d weights in groups of %d (64, a power of two)", qblock, qblock2);
  if (n_tokens < 0 || n_tokens > kGemvTokens || rows < 1 || rows > (1 << 30) || cols < 64 || cols % 64 ||
      cols > (1 << 24) || ldx < cols || ldx % 8 || ldx > (1 << 24) || ldo < rows)
    return fail(TALM_EINVAL,
                "nf4_gemv: bad shape (tokens %lld, W [%lld, %lld], ldx %lld, ldo %lld): at most %d tokens, cols "
                "a multiple of 64, ldx of 8",
                (long long)n_tokens, (long long)rows, (long long)cols, (long long)ldx, (long long)ldo, kGemvTokens);
  if (ts && (ldt < (b1 ? 32 : 16) || !b0 || lo0 < 0 || hi0 < lo0 || hi0 > rows ||
             (b1 && (lo1 < 0 || hi1 < lo1 || hi1 > rows))))
    return fail(TALM_EINVAL, "nf4_gemv: adapters on rows %lld..%lld / %lld..%lld, ldt %lld", (long long)lo0,
                (long long)hi0, (long long)lo1, (long long)hi1, (long long)ldt);
  if (n_tokens == 0) return ok();
  if (!x || !packed || !absmax8 || !code || !absmax2 || !offset2 || !out)
    return fail(TALM_EINVAL, "nf4_gemv: null pointer");
  if (!aligned(x, 16) || !aligned(packed, 16)) return fail(TALM_EINVAL, "nf4_gemv: x and packed 16-byte aligned");
  GemvArgs a{};
  a.x = x; a.ldx = ldx; a.M = static_cast<int>(n_tokens);
  a.rows = static_cast<int>(rows); a.cols = static_cast<int>(cols);
  a.packed = packed; a.absmax8 = absmax8; a.code = code; a.absmax2 = absmax2; a.offset2 = offset2;
  while ((1 << a.shift2) < qblock2) ++a.shift2;
  a.bias = bias; a.out = out; a.ldo = ldo;
  if (ts) {
    a.ts = ts; a.ldt = ldt;
    a.b[0] = b0; a.lo[0] = static_cast<int>(lo0); a.hi[0] = static_cast<int>(hi0);
    if (b1) { a.b[1] = b1; a.lo[1] = static_cast<int>(lo1); a.hi[1] = static_cast<int>(hi1); }
  }
  // The table in LDS pays from some size of W on, an earlier one with more tokens. us, rows / lut:
  // 1 token [1536, 4864] 5.0 / 5.3, [8960, 1024] 5.1 / 5.2, [8960, 1536] 7.2 / 6.0; 16 tokens [4864, 896]
  // 4.6 / 5.2, [1536, 3584] 7.9 / 6.0, [1536, 4864] 9.7 / 6.8; 32 tokens [2048, 1536] 6.1 / 6.1,
  // [1792, 2048] 7.1 / 6.0, [1536, 3584] 11.5 / 7.5.
  const bool lut = rows * cols > (n_tokens <= 8 ? 9 << 20 : n_tokens <= 16 ? 5 << 20 : 3 << 20);
  // Parts of the reduction per tile: what the tokens leave room for, and
  //   rows kernel: the fewest idle lanes and CUs (1 token, one / two / four parts: [2048, 1536] 3.8 / 3.2 /
  //     3.8 us, [4864, 896] 3.7 / 3.8 / 4.0);
  //   lut kernel: two where whole tiles would leave CUs without one (1 token, one / two parts: [1536, 8960]
  //     8.3 / 6.8, [2048, 8192] 8.2 / 6.2), of 9 tokens on, which then are two blocks, where the halves
  //     leave no CU with two (16 tokens: [2048, 8192] 10.3 / 8.6; [3584, 18944] 20 / 27).
  int best = 1;
  const double cus = device_cus();
  if (lut) {
    const int64_t tiles = (rows + 15) / 16;
    best = n_tokens <= 8 ? (tiles < device_cus() ? 2 : 1) : (n_tokens <= 16 && 2 * tiles <= device_cus() ? 2 : 1);
  } else {
    double cost = 0;
    for (int p = 1; p <= 4 && p * n_tokens <= 16; p *= 2) {
      const int64_t units = (cols + 256 * p - 1) / (256 * p), wgs = (rows * p + 15) / 16;
      const double waste = static_cast<double>(units * 256 * p) / cols;
      const double c = waste * std::max(1.0, cus / static_cast<double>(wgs));
      if (cost == 0 || c < cost) { cost = c; best = p; }
    }
  }
  const hipStream_t s = as_stream(stream);
  if (lut) {
    if (n_tokens > 16) launch_lut_form<1, 2>(a, s);
    else if (best == 1) launch_lut_form<1, 1>(a, s);
    else if (n_tokens > 8) launch_lut_form<2, 2>(a, s);
    else launch_lut_form<2, 1>(a, s);
  } else if (n_tokens > 16) {
    launch_rows<1, 2>(a, s);
  } else if (best == 1) {
    launch_rows<1, 1>(a, s);
  } else if (best == 2) {
    launch_rows<2, 1>(a, s);
  } else {
    launch_rows<4, 1>(a, s);
  }
  return check_launch("nf4_gemv");
}
