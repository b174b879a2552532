// Dropout and the LoRA adapters' products with dropout on their input, for gfx950. No mask is
// stored: every kernel computes it from the generator (philox.h).
//
//   dropout          y = keep x factor                      (the gradient: the same on dy)
//   lora_down_drop   t = factor (keep x) A^T, ts = s t      (rank 16; 1 or 2 adapters of one x, each
//                                                            with a mask of its own)
//   lora_branch_fwd  t, then y = s t B^T                    (one adapter)
//   lora_bwd_drop    dA_g = factor u_g^T (keep_g x), dB_g = s_g dy_g^T t_g,
//                    dx = base + sum_g factor keep_g (u_g A_g)
// The adapters' arithmetic is PEFT's (solution/lora.py:183-231, solution/fused_proj.py:139-153,
// :188-215) with x / (1 - p) not rounded on the way: the mask clears fp16 operands exactly and the
// factor goes on the fp32 sums.
//
// t and u enter their second products in fp16, like every MFMA operand: as the reference's adapters keep them
// under autocast. Relative L2 of the gradients against 64 bits 2.9e-4, 2.1e-4 from the results' rounding alone.
//
// An adapter of 8960 inputs and 1536 outputs on 2048 tokens, us (MI355X): down 13.2, up 5.0; u 5.6 (the plain
// down product on dy), backward 21.7, its sums 4.2: 50 for 124 MB that have to move (25 at 4.93 TB/s). On 1312 tokens
// of 1536 inputs: 4.3, 3.7, 5.6, 8.2, 3.0.
// In a packed layer (lora_down_drop, lora_bwd_drop onto the base product's dx, its sums included): q and v of 1312
// tokens, two masks of x, down 7.6, u 5.2, backward 15.6; of 2048 tokens 7.7, 5.2, 20.3; down_proj's 8960 inputs on
// 2048 tokens 18.5 (lora_down_drop does not split its reduction), 4.9, 31.9.
#include "mfma_tile.h"
#include "philox.h"

#include <algorithm>

namespace talm {
namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint16_t half4_t __attribute__((ext_vector_type(4)));

constexpr int kRank = 16;
constexpr int kMaxAdapters = 2;

__device__ __forceinline__ half8_t h8(uint4 v) { return __builtin_bit_cast(half8_t, v); }

// ------------------------------------------------------------------------------------------
// Elementwise
// ------------------------------------------------------------------------------------------
struct F16Elem {
  static __device__ __forceinline__ float get(uint16_t v) { return h2f(v); }
  static __device__ __forceinline__ uint16_t put(float v) { return f2h(v); }
  typedef uint16_t type;
};
struct BF16Elem {
  static __device__ __forceinline__ float get(uint16_t v) {
    return __builtin_bit_cast(float, static_cast<uint32_t>(v) << 16);
  }
  static __device__ __forceinline__ uint16_t put(float v) {
    return __builtin_bit_cast(uint16_t, static_cast<__bf16>(v));
  }
  typedef uint16_t type;
};
struct F32Elem {
  static __device__ __forceinline__ float get(float v) { return v; }
  static __device__ __forceinline__ float put(float v) { return v; }
  typedef float type;
};

// n / d of n < 2^31 as (mulhi(mul, n) + n) >> shift; shift -1: the division itself.
struct Divider {
  uint32_t mul;
  int shift;
};
Divider divider(int64_t most, int64_t d) {
  if (most >= int64_t{1} << 31) return Divider{0, -1};
  int s = 0;
  while ((int64_t{1} << s) < d) ++s;
  return Divider{static_cast<uint32_t>((((uint64_t{1} << s) - d) << 32) / d + 1), s};
}

// One thread per eight columns of a row, `first` those of the launches before. kVec: whole chunks, 16-byte
// aligned rows. The generator, about 70 VALU instructions per chunk with 20 of them at a quarter of the rate,
// runs beside other wavefronts' loads: the thread's own load is issued before the key's (the other way round
// bf16 [2048, 8960] took 16.8 us for 14.2).
// Bound by memory: bf16 [2048, 8960] 13.4 us (5.5 TB/s) with four x and y in turn, 12.2 (6.0) where one pair stays
// in the last-level cache, [40000, 4096] 107 (6.1; a large copy reaches 4.9); fp32 [2048, 8960] 31.1 (4.7), 23.9.
template <class E, bool kVec>
__global__ __launch_bounds__(256) void dropout_kernel(const typename E::type* __restrict__ x, int64_t ldx,
                                                      int64_t rows, int64_t cols, float factor,
                                                      DropArgs drop, typename E::type* __restrict__ y,
                                                      int64_t ldy, int64_t first, Divider div) {
  typedef typename E::type T;
  const int64_t per_row = (cols + 7) / 8;
  const int64_t block = first + static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  if (block >= rows * per_row) return;
  int64_t r;
  if (div.shift >= 0) {
    const uint32_t n = static_cast<uint32_t>(block);
    r = (__umulhi(div.mul, n) + n) >> div.shift;
  } else {
    r = block / per_row;
  }
  const int64_t c = (block - r * per_row) * 8;
  const T* xp = x + r * ldx + c;
  T* yp = y + r * ldy + c;
  const int n = kVec ? 8 : static_cast<int>(min(cols - c, static_cast<int64_t>(8)));
  T v[8];
  if constexpr (kVec) {
    *reinterpret_cast<uint4*>(v) = *reinterpret_cast<const uint4*>(xp);
    if constexpr (sizeof(T) == 4) *reinterpret_cast<uint4*>(v + 4) = *reinterpret_cast<const uint4*>(xp + 4);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = e < n ? xp[e] : T(0);
  }
  const DropKey key(drop.key, drop.site, drop.threshold);
  const uint4 bits = philox_block(static_cast<uint64_t>(block), key);
  const uint32_t w[4] = {bits.x, bits.y, bits.z, bits.w};
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const uint32_t u = e & 1 ? w[e >> 1] >> 16 : w[e >> 1] & 0xffffu;
    v[e] = u >= key.threshold ? E::put(E::get(v[e]) * factor) : T(0);
  }
  if constexpr (kVec) {
    *reinterpret_cast<uint4*>(yp) = *reinterpret_cast<const uint4*>(v);
    if constexpr (sizeof(T) == 4) *reinterpret_cast<uint4*>(yp + 4) = *reinterpret_cast<const uint4*>(v + 4);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (e < n) yp[e] = v[e];
  }
}

// ------------------------------------------------------------------------------------------
// t = factor (keep x) A^T
// ------------------------------------------------------------------------------------------
struct DownArgs {
  const uint16_t* x;  // [N][ldx]
  int64_t ldx;
  int n_tokens, k, n_adapters, parts;
  const uint16_t* a[kMaxAdapters];  // [16][k]
  float scaling[kMaxAdapters];
  float factor;
  DropArgs drop;
  uint32_t site[kMaxAdapters];
  uint16_t* t;                  // [N][ldt], 16 columns per adapter
  uint16_t* ts;
  int64_t ldt;
  float* part;                  // one adapter's sums [parts][N][16] instead (no factor), or null
};

constexpr int kDownWaves = 8;
constexpr int kDownBatch = 4;
constexpr int kDownMaxParts = 4;
constexpr int64_t kDownCus = 256;  // the chip's CUs, for plans that a size query makes without a device

// One workgroup per 16 tokens and part of the reduction; its wavefronts take the part's 32-deep
// steps round-robin, the loads of kDownBatch of them before their MFMAs. Bound by the generator: 2.3 million
// blocks of x [2048, 8960] take the VALU about 7.6 of the 13.2 us, the 37 MB of x as long (4.93 TB/s), half
// behind each other (not kept, no faster: two adjacent steps per wavefront; the next batch's loads
// ahead of this one's masks). The reduction in one part, as talm_lora_down_drop runs it: 18.5 us.
template <int G>
__global__ __launch_bounds__(64 * kDownWaves) void lora_down_drop_kernel(DownArgs a) {
  __shared__ float red[kDownWaves][G][16][16 + 1];
  const int m0 = blockIdx.x * 16;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int row = lane & 15, kq = 8 * (lane >> 4);
  const int steps = a.k >> 5, per = (steps + a.parts - 1) / a.parts;
  const int s_lo = blockIdx.y * per, s_hi = min(steps, s_lo + per);
  const __amdgpu_buffer_rsrc_t rx = buffer_rsrc(a.x + static_cast<int64_t>(m0) * a.ldx);
  const uint32_t xoff = m0 + row < a.n_tokens ? static_cast<uint32_t>((row * a.ldx + kq) * 2) : kOob;
  const uint32_t aoff = static_cast<uint32_t>((row * a.k + kq) * 2);
  const uint64_t block0 = static_cast<uint64_t>(m0 + row) * (a.k >> 3) + (kq >> 3);
  f32x4 acc[G];
#pragma unroll
  for (int g = 0; g < G; ++g) acc[g] = f32x4{0.f, 0.f, 0.f, 0.f};
  const DropKey key(a.drop.key, 0, a.drop.threshold);
  for (int base = s_lo + wave; base < s_hi; base += kDownWaves * kDownBatch) {
    uint4 xv[kDownBatch], av[kDownBatch][G];
#pragma unroll
    for (int j = 0; j < kDownBatch; ++j) {
      const int c = base + kDownWaves * j;
      const bool live = c < s_hi;
      const uint32_t kb = static_cast<uint32_t>(c) * 64;
      xv[j] = __builtin_bit_cast(uint4, __builtin_amdgcn_raw_buffer_load_b128(rx, live ? xoff + kb : kOob, 0, 0));
#pragma unroll
      for (int g = 0; g < G; ++g)
        av[j][g] = __builtin_bit_cast(
            uint4, __builtin_amdgcn_raw_buffer_load_b128(buffer_rsrc(a.a[g]), live ? aoff + kb : kOob, 0, 0));
    }
#pragma unroll
    for (int j = 0; j < kDownBatch; ++j) {
      if (base + kDownWaves * j >= s_hi) break;
      const uint64_t block = block0 + static_cast<uint64_t>(base + kDownWaves * j) * 4;
#pragma unroll
      for (int g = 0; g < G; ++g) {
        DropKey kg = key;
        kg.site = a.site[g];
        const uint4 xd = key.threshold ? keep8(xv[j], philox_block(block, kg), key.threshold) : xv[j];
        acc[g] = __builtin_amdgcn_mfma_f32_16x16x32_f16(h8(xd), h8(av[j][g]), acc[g], 0, 0, 0);
      }
    }
  }
  // accumulator element v of lane l: token 4 (l / 16) + v, rank l % 16
#pragma unroll
  for (int g = 0; g < G; ++g)
#pragma unroll
    for (int v = 0; v < 4; ++v) red[wave][g][4 * (lane >> 4) + v][lane & 15] = acc[g][v];
  __syncthreads();
  for (int e = threadIdx.x; e < G * 256; e += 64 * kDownWaves) {
    const int g = e >> 8, r = (e >> 4) & 15, i = e & 15;
    if (m0 + r >= a.n_tokens) continue;
    float sum = 0.f;
#pragma unroll
    for (int w = 0; w < kDownWaves; ++w) sum += red[w][g][r][i];
    if (G == 1 && a.part) {
      a.part[(static_cast<int64_t>(blockIdx.y) * a.n_tokens + m0 + r) * kRank + i] = sum;
    } else {
      const int64_t at = static_cast<int64_t>(m0 + r) * a.ldt + g * kRank + i;
      a.t[at] = f2h(a.factor * sum);
      a.ts[at] = f2h(a.scaling[g] * (a.factor * sum));
    }
  }
}

// ------------------------------------------------------------------------------------------
// y = s t B^T, t = factor times the parts of the down product
// ------------------------------------------------------------------------------------------
struct UpArgs {
  const float* part;  // [parts][N][16]
  int parts, n_tokens, cols;
  float factor, scaling;
  uint16_t* t;        // [N][16]: what the backward keeps
  const uint16_t* b;  // [cols][16]
  uint16_t* y;        // [N][cols]
};

constexpr int kUpTokens = 64;  // per workgroup, in blocks of 32

// Column of a 32-column block that row m of the A operand holds, so that a lane's 16 accumulators (rows
// 8 (v / 4) + 4 (lane / 32) + v % 4) are the 16 consecutive columns 16 (lane / 32) .. + 15.
__device__ __forceinline__ int up_column(int m) { return 16 * ((m >> 2) & 1) + 4 * (m >> 3) + (m & 3); }

// One wavefront per 32 columns: C[c][token] = B t^T (v_mfma_f32_32x32x16_f16, K = the rank), a lane owns
// a token and 16 consecutive columns: two 16-byte stores. The parts (at most kDownMaxParts) are summed
// here, in order, by every workgroup that reads them: one launch less than a sum of their own. Bound by
// latency: 2.5 us above a launch for 2048 tokens, 6 MB written.
__global__ __launch_bounds__(256) void lora_up_kernel(UpArgs a) {
  const int lane = threadIdx.x & 63, hh = lane >> 5, l32 = lane & 31;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int c0 = blockIdx.x * 128 + 32 * wave;
  if (c0 >= a.cols) return;  // no barrier follows
  const int cm = min(c0 + up_column(l32), a.cols - 1), col = c0 + 16 * hh;
  const uint4 bf = *reinterpret_cast<const uint4*>(a.b + static_cast<int64_t>(cm) * kRank + 8 * hh);
#pragma unroll
  for (int tb = 0; tb < kUpTokens / 32; ++tb) {
    const int tok = blockIdx.y * kUpTokens + 32 * tb + l32;
    const bool in = tok < a.n_tokens;
    const float* p = a.part + static_cast<int64_t>(in ? tok : a.n_tokens - 1) * kRank + 8 * hh;
    // every part's loads before their adds: a part past the last is the last one again, its bits cleared
    // (a product with 0 would turn an infinity into NaN; a select would be a branch before the loads)
    float4 lo[kDownMaxParts], hi[kDownMaxParts];
#pragma unroll
    for (int i = 0; i < kDownMaxParts; ++i) {
      const float* q = p + static_cast<int64_t>(min(i, a.parts - 1)) * a.n_tokens * kRank;
      lo[i] = reinterpret_cast<const float4*>(q)[0];
      hi[i] = reinterpret_cast<const float4*>(q)[1];
    }
    float s[8] = {lo[0].x, lo[0].y, lo[0].z, lo[0].w, hi[0].x, hi[0].y, hi[0].z, hi[0].w};
#pragma unroll
    for (int i = 1; i < kDownMaxParts; ++i) {
      const uint32_t is = i < a.parts ? 0xffffffffu : 0u;
      const float v[8] = {lo[i].x, lo[i].y, lo[i].z, lo[i].w, hi[i].x, hi[i].y, hi[i].z, hi[i].w};
#pragma unroll
      for (int e = 0; e < 8; ++e) s[e] += __builtin_bit_cast(float, __builtin_bit_cast(uint32_t, v[e]) & is);
    }
    const float f = a.factor;
    const uint4 tf = make_uint4(pack2(f * s[0], f * s[1]), pack2(f * s[2], f * s[3]), pack2(f * s[4], f * s[5]),
                                pack2(f * s[6], f * s[7]));
    if (c0 == 0 && in) *reinterpret_cast<uint4*>(a.t + static_cast<int64_t>(tok) * kRank + 8 * hh) = tf;
    f32x16 acc;
#pragma unroll
    for (int v = 0; v < 16; ++v) acc[v] = 0.f;
    acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(h8(bf), h8(tf), acc, 0, 0, 0);
    if (!in) continue;
#pragma unroll
    for (int q = 0; q < 2; ++q)
      if (col + 8 * q < a.cols) {
        float v[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = a.scaling * acc[8 * q + e];
        *reinterpret_cast<uint4*>(a.y + static_cast<int64_t>(tok) * a.cols + col + 8 * q) =
            make_uint4(pack2(v[0], v[1]), pack2(v[2], v[3]), pack2(v[4], v[5]), pack2(v[6], v[7]));
      }
  }
}

// ------------------------------------------------------------------------------------------
// dA_g = factor u_g^T (keep_g x), dB_g = s_g dy_g^T t_g, dx = base + sum_g factor keep_g (u_g A_g)
// ------------------------------------------------------------------------------------------
struct BwdArgs {
  const uint16_t* x;
  int64_t ldx;
  const uint16_t* dy;
  int64_t ldy;
  const uint16_t* u;  // [N][ldu], 16 columns per adapter
  int64_t ldu;
  const uint16_t* t;
  int64_t ldt;
  int n_tokens, hidden, n_adapters;
  int lo[kMaxAdapters], seg[kMaxAdapters];
  float scaling[kMaxAdapters], factor;
  DropArgs drop;
  uint32_t site[kMaxAdapters];
  const uint16_t* a[kMaxAdapters];  // [16][hidden]: for dx
  const uint16_t* base;             // [N][ldb] or null
  int64_t ldb;
  uint16_t* dx;                     // [N][ldd] or null; may be base
  int64_t ldd;
  // the reductions' columns one after the other: dA of each adapter, then dB of each, every one
  // padded to whole workgroups of 128
  int first[2 * kMaxAdapters + 1];
  int cols;             // first[2 n_adapters]
  int chunk, chunks;    // tokens per partial (a multiple of 64), partials
  float* part;          // [chunks][cols][16]
  int half_out;         // the gradients in fp16, else fp32
  void* da[kMaxAdapters];
  void* db[kMaxAdapters];
};

constexpr int kBwTok = 64;
constexpr int kBwLd = 128 + 16;  // halves per staged row: rows 32 bytes apart in the banks

// See read_tr_untracked of attn.hip: lane i of a group of 16 gets elements 0..3 = rows 0..3 of column i
// of the 4 x 16 block whose row j / 4, columns 4 (j % 4) .. + 3 lane j points at.
__device__ __forceinline__ half4_t read_tr(const uint16_t* p) {
  const auto r = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4_ptr)(p));
  return __builtin_bit_cast(half4_t, r);
}
__device__ __forceinline__ half8_t pair(half4_t lo, half4_t hi) {
  return __builtin_bit_cast(half8_t, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
}

// One workgroup per (128 columns, chunk of tokens); columns of x for every adapter, or of one adapter's
// dy. 64 tokens at a time: the rows staged in LDS (x under each adapter's mask, computed once for the
// weight gradient and dx), the next tokens' loads in flight meanwhile. Weight gradients: the fragments
// read transposed, each wavefront 32 columns against the 16 of u or t (v_mfma_f32_16x16x32_f16). dx:
// each wavefront 32 columns, C[c][token] = A^T u^T as in lora_up_kernel, its A fragment gathered once.
// One pass over x for both gradients and one computation of its mask: 21.7 us at [2048, 8960] with 1536
// output columns, 91 MB with the partials, 4.2 TB/s (two kernels with the mask computed twice: 15 and 14).
template <int G>
__global__ __launch_bounds__(256) void lora_bwd_drop_kernel(BwdArgs a) {
  __shared__ __attribute__((aligned(16))) uint16_t xs[G][kBwTok][kBwLd];
  __shared__ __attribute__((aligned(16))) uint16_t ms[G][kBwTok][kRank + 8];
  __shared__ __attribute__((aligned(16))) uint8_t bits[G][kBwTok][16];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  // x's column blocks come first (first[1] is one adapter's width), then each adapter's dy
  const int x_blocks = a.first[1] >> 7;
  const bool is_b = static_cast<int>(blockIdx.x) >= x_blocks;
  int job = 0, c0 = blockIdx.x * 128;  // the reduction, and its first column here
  if (is_b) {
    c0 += (G - 1) * a.first[1];
    job = G;
    while (job + 1 < 2 * G && c0 >= a.first[job + 1]) ++job;
  }
  const int gb = is_b ? job - G : 0;       // the adapter of a dB block
  const int n_g = is_b ? 1 : G;
  const int cb = c0 - a.first[job];
  const int width = is_b ? a.seg[gb] : a.hidden;
  const uint16_t* src = is_b ? a.dy + a.lo[gb] : a.x;
  const int64_t ld = is_b ? a.ldy : a.ldx;
  const uint16_t* mat = is_b ? a.t + kRank * gb : a.u;
  const int64_t ldm = is_b ? a.ldt : a.ldu;
  const uint32_t threshold = is_b ? 0u : a.drop.threshold;
  const DropKey key(a.drop.key, 0, threshold);
  const int r_lo = blockIdx.y * a.chunk, r_hi = min(a.n_tokens, r_lo + a.chunk);
  // a thread's items: 16-byte chunk tid % 16 of rows tid / 16 + 16 i; of u / t threads 0..127 one chunk
  const int cc = cb + 8 * (tid & 15);
  const bool live = cc < width;
  const uint4 zero = make_uint4(0u, 0u, 0u, 0u);
  uint4 xv[4], mv[G];
  auto load = [&](int r0) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int r = r0 + (tid >> 4) + 16 * i;
      xv[i] = zero;
      if (live && r < r_hi) xv[i] = *reinterpret_cast<const uint4*>(src + static_cast<int64_t>(r) * ld + cc);
    }
    const int r = r0 + (tid >> 1);
#pragma unroll
    for (int g = 0; g < G; ++g) {
      mv[g] = zero;
      if (g < n_g && tid < 128 && r < r_hi)
        mv[g] = *reinterpret_cast<const uint4*>(mat + static_cast<int64_t>(r) * ldm + kRank * g + 8 * (tid & 1));
    }
  };
  // dx: the adapters' A fragments, lane row l % 32 the column up_column of the wavefront's 32
  const int l32 = lane & 31, hh = lane >> 5;
  const bool has_dx = !is_b && a.dx != nullptr;
  uint4 af[G];
#pragma unroll
  for (int g = 0; g < G; ++g) {
    af[g] = zero;
    const int c = cb + 32 * wave + up_column(l32);
    if (has_dx && c < a.hidden) {
      uint32_t h[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) h[e] = a.a[g][static_cast<int64_t>(8 * hh + e) * a.hidden + c];
      af[g] = make_uint4(h[0] | h[1] << 16, h[2] | h[3] << 16, h[4] | h[5] << 16, h[6] | h[7] << 16);
    }
  }
  f32x4 acc[G][2];
#pragma unroll
  for (int g = 0; g < G; ++g) acc[g][0] = acc[g][1] = f32x4{0.f, 0.f, 0.f, 0.f};
  load(r_lo);
  const int grp = lane >> 4, j = lane & 15;
  for (int r0 = r_lo; r0 < r_hi; r0 += kBwTok) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int r = (tid >> 4) + 16 * i;
#pragma unroll
      for (int g = 0; g < G; ++g) {
        if (g >= n_g) break;
        uint4 v = xv[i];
        if (threshold) {
          DropKey kg = key;
          kg.site = a.site[g];
          const uint4 rnd = philox_block(static_cast<uint64_t>(r0 + r) * (a.hidden >> 3) + (cc >> 3), kg);
          v = keep8(v, rnd, threshold);
          if (has_dx) bits[g][r][tid & 15] = static_cast<uint8_t>(keep_bits(rnd, threshold));
        }
        *reinterpret_cast<uint4*>(&xs[g][r][8 * (tid & 15)]) = v;
      }
    }
    if (tid < 128)
#pragma unroll
      for (int g = 0; g < G; ++g) *reinterpret_cast<uint4*>(&ms[g][tid >> 1][8 * (tid & 1)]) = mv[g];
    __syncthreads();
    if (r0 + kBwTok < r_hi) load(r0 + kBwTok);
    if (has_dx) {
      const int lc = 32 * wave + 16 * hh, col = cb + lc;  // the lane's 16 columns
#pragma unroll
      for (int tb = 0; tb < kBwTok / 32; ++tb) {
        const int rl = 32 * tb + l32, tok = r0 + rl;
        float sum[16];
#pragma unroll
        for (int e = 0; e < 16; ++e) sum[e] = 0.f;
        if (a.base && tok < r_hi)
#pragma unroll
          for (int q = 0; q < 2; ++q)
            if (col + 8 * q < a.hidden) {
              const uint4 b = *reinterpret_cast<const uint4*>(a.base + static_cast<int64_t>(tok) * a.ldb + col + 8 * q);
              const uint32_t w[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                sum[8 * q + 2 * e] = lo_f(w[e]);
                sum[8 * q + 2 * e + 1] = hi_f(w[e]);
              }
            }
#pragma unroll
        for (int g = 0; g < G; ++g) {
          const uint4 uf = *reinterpret_cast<const uint4*>(&ms[g][rl][8 * hh]);
          f32x16 d;
#pragma unroll
          for (int v = 0; v < 16; ++v) d[v] = 0.f;
          d = __builtin_amdgcn_mfma_f32_32x32x16_f16(h8(af[g]), h8(uf), d, 0, 0, 0);
          uint32_t keep = 0xffffu;
          if (threshold) keep = *reinterpret_cast<const uint16_t*>(&bits[g][rl][lc >> 3]);
#pragma unroll
          for (int e = 0; e < 16; ++e) sum[e] += keep >> e & 1 ? a.factor * d[e] : 0.f;
        }
        if (tok < r_hi)
#pragma unroll
          for (int q = 0; q < 2; ++q)
            if (col + 8 * q < a.hidden) {
              const float* s = sum + 8 * q;
              *reinterpret_cast<uint4*>(a.dx + static_cast<int64_t>(tok) * a.ldd + col + 8 * q) =
                  make_uint4(pack2(s[0], s[1]), pack2(s[2], s[3]), pack2(s[4], s[5]), pack2(s[6], s[7]));
            }
      }
    }
#pragma unroll
    for (int ks = 0; ks < kBwTok / 32; ++ks) {
      const int k0 = 32 * ks + 8 * grp + (j >> 2);  // the lane's row of the first transposed read
#pragma unroll
      for (int g = 0; g < G; ++g) {
        if (g >= n_g) break;
        const half8_t mb = pair(read_tr(&ms[g][k0][4 * (j & 3)]), read_tr(&ms[g][k0 + 4][4 * (j & 3)]));
#pragma unroll
        for (int b = 0; b < 2; ++b) {
          const int c = 32 * wave + 16 * b + 4 * (j & 3);
          acc[g][b] = __builtin_amdgcn_mfma_f32_16x16x32_f16(pair(read_tr(&xs[g][k0][c]), read_tr(&xs[g][k0 + 4][c])),
                                                            mb, acc[g][b], 0, 0, 0);
        }
      }
    }
    __syncthreads();
  }
#pragma unroll
  for (int g = 0; g < G; ++g) {
    if (g >= n_g) break;
    float* out = a.part + (static_cast<int64_t>(blockIdx.y) * a.cols + c0 + g * a.first[1] + 32 * wave) * kRank;
#pragma unroll
    for (int b = 0; b < 2; ++b)
#pragma unroll
      for (int v = 0; v < 4; ++v) out[(16 * b + 4 * grp + v) * kRank + j] = acc[g][b][v];
  }
}

// The chunks summed in order: one thread per (column, rank).
__global__ __launch_bounds__(256) void lora_wgrad_sum_kernel(BwdArgs a) {
  const int64_t e = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  if (e >= static_cast<int64_t>(a.cols) * kRank) return;
  const int c = static_cast<int>(e / kRank), i = static_cast<int>(e % kRank);
  int job = 0;
  while (job + 1 < 2 * a.n_adapters && c >= a.first[job + 1]) ++job;
  const bool is_b = job >= a.n_adapters;
  const int g = is_b ? job - a.n_adapters : job, cj = c - a.first[job];
  if (cj >= (is_b ? a.seg[g] : a.hidden)) return;
  const int64_t step = static_cast<int64_t>(a.cols) * kRank;
  float sum = 0.f;
  for (int k0 = 0; k0 < a.chunks; k0 += 8) {
    float v[8];  // eight loads before their adds (selects, so that none is sunk to its add)
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = a.part[min(k0 + k, a.chunks - 1) * step + e];
#pragma unroll
    for (int k = 0; k < 8; ++k) sum += k0 + k < a.chunks ? v[k] : 0.f;
  }
  const float v = (is_b ? a.scaling[g] : a.factor) * sum;
  const int64_t at = is_b ? static_cast<int64_t>(cj) * kRank + i : static_cast<int64_t>(i) * a.hidden + cj;
  void* out = is_b ? a.db[g] : a.da[g];
  if (a.half_out) static_cast<uint16_t*>(out)[at] = f2h(v);
  else static_cast<float*>(out)[at] = v;
}

bool fits32(int64_t rows, int64_t ld) { return rows * ld * 2 < (int64_t{1} << 31); }

int check_drop(const char* what, const int64_t* key, float p) {
  if (!(p >= 0.f && p < 1.f)) return fail(TALM_EINVAL, "%s: p %g (0 <= p < 1)", what, static_cast<double>(p));
  if (drop_threshold(p) && !key) return fail(TALM_EINVAL, "%s: p %g without a key", what, static_cast<double>(p));
  if (!aligned(key, 8)) return fail(TALM_EINVAL, "%s: the key must be 8-byte aligned", what);
  return TALM_OK;
}

// Parts of the branch's down product: about two workgroups per CU, at least two 32-deep steps for each
// of a workgroup's wavefronts.
int down_parts(int64_t n_tokens, int64_t k) {
  const int64_t blocks = std::max<int64_t>(1, (n_tokens + 15) / 16), steps = k / 32;
  const int64_t most = std::min<int64_t>(kDownMaxParts, steps / (2 * kDownWaves));
  return static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(most, 2 * kDownCus / blocks)));
}

struct BwdPlan {
  int64_t cols = 0, x_blocks = 0, chunk = 0, chunks = 0;
};
BwdPlan bwd_plan(int64_t n_tokens, int64_t hidden, int64_t n_adapters, int64_t seg0, int64_t seg1) {
  auto pad = [](int64_t n) { return (n + 127) / 128 * 128; };
  BwdPlan w;
  w.x_blocks = pad(hidden) / 128;
  w.cols = n_adapters * pad(hidden) + pad(seg0) + (n_adapters > 1 ? pad(seg1) : 0);
  // 128 tokens to a partial while that gives the chip three rounds of workgroups at most, whole multiples
  // of it from there on: fewer partials to write and sum
  const int64_t blocks = w.cols / 128 - (n_adapters - 1) * w.x_blocks;
  w.chunk = 128 * std::max<int64_t>(1, (n_tokens + 127) / 128 * blocks / (3 * kDownCus));
  w.chunks = std::max<int64_t>(1, (n_tokens + w.chunk - 1) / w.chunk);
  return w;
}

}  // namespace
}  // namespace talm

using namespace talm;

TALM_API int talm_dropout(const void* x, int64_t ldx, int64_t rows, int64_t cols, int32_t dtype, float p,
                          const int64_t* key, uint32_t site, void* y, int64_t ldy, void* stream) {
  if (rows < 0 || cols < 0 || ldx < cols || ldy < cols ||
      (cols > 0 && rows > (int64_t{1} << 38) / ((cols + 7) / 8)))
    return fail(TALM_EINVAL, "dropout: bad shape (%lld x %lld, row strides %lld / %lld)", (long long)rows,
                (long long)cols, (long long)ldx, (long long)ldy);
  if (dtype != TALM_F32 && dtype != TALM_F16 && dtype != TALM_BF16)
    return fail(TALM_EINVAL, "dropout: dtype %d", dtype);
  const int status = check_drop("dropout", key, p);
  if (status != TALM_OK) return status;
  if (rows == 0 || cols == 0) return ok();
  if (!x || !y) return fail(TALM_EINVAL, "dropout: null pointer");
  const DropArgs drop{key, site, drop_threshold(p)};
  const float factor = drop_factor(drop.threshold);
  const int64_t n = rows * ((cols + 7) / 8);
  const Divider div = divider(n, (cols + 7) / 8);
  const int64_t unit = dtype == TALM_F32 ? 4 : 8;  // elements of 16 bytes
  const bool vec = cols % 8 == 0 && ldx % unit == 0 && ldy % unit == 0 && aligned(x, 16) && aligned(y, 16);
  const hipStream_t s = as_stream(stream);
#define TALM_DROPOUT(E, V)                                                                             \
  hipLaunchKernelGGL((dropout_kernel<E, V>), grid, dim3(256), 0, s, static_cast<const E::type*>(x), ldx, \
                     rows, cols, factor, drop, static_cast<E::type*>(y), ldy, first, div)
  constexpr int64_t kMost = int64_t{1} << 30;  // a launch's threads stay below 2^32
  for (int64_t first = 0; first < n; first += kMost) {
    const dim3 grid(static_cast<unsigned>((std::min(kMost, n - first) + 255) / 256));
    if (dtype == TALM_F32) { if (vec) TALM_DROPOUT(F32Elem, true); else TALM_DROPOUT(F32Elem, false); }
    else if (dtype == TALM_F16) { if (vec) TALM_DROPOUT(F16Elem, true); else TALM_DROPOUT(F16Elem, false); }
    else { if (vec) TALM_DROPOUT(BF16Elem, true); else TALM_DROPOUT(BF16Elem, false); }
  }
#undef TALM_DROPOUT
  return check_launch("dropout");
}

namespace talm {
namespace {

void launch_down(const DownArgs& a, hipStream_t s) {
  const dim3 grid(static_cast<unsigned>((a.n_tokens + 15) / 16), static_cast<unsigned>(a.parts));
  if (a.n_adapters > 1) hipLaunchKernelGGL(lora_down_drop_kernel<2>, grid, dim3(64 * kDownWaves), 0, s, a);
  else hipLaunchKernelGGL(lora_down_drop_kernel<1>, grid, dim3(64 * kDownWaves), 0, s, a);
}

}  // namespace
}  // namespace talm

TALM_API int talm_lora_down_drop(const uint16_t* x, int64_t ldx, int64_t n_tokens, int64_t k,
                                 const uint16_t* a0, const uint16_t* a1, int32_t n_adapters, float p,
                                 const int64_t* key, uint32_t site0, uint32_t site1, float scaling0,
                                 float scaling1, uint16_t* t, uint16_t* ts, int64_t ldt, void* stream) {
  const bool two = n_adapters > 1;
  if (n_tokens < 0 || n_tokens > (1 << 30) || n_adapters < 1 || n_adapters > kMaxAdapters || k < 32 || k % 32 ||
      ldx < k || ldx % 8 || ldt < kRank * n_adapters || !fits32(16, ldx) || !fits32(16, k))
    return fail(TALM_EINVAL,
                "lora_down_drop: bad shape (tokens %lld, k %lld, ldx %lld, adapters %d, ldt %lld): k a "
                "multiple of 32 inside x's rows of a multiple of 8, 1-2 adapters of rank 16",
                (long long)n_tokens, (long long)k, (long long)ldx, n_adapters, (long long)ldt);
  const int status = check_drop("lora_down_drop", key, p);
  if (status != TALM_OK) return status;
  if (n_tokens == 0) return ok();
  if (!x || !a0 || (two && !a1) || !t || !ts) return fail(TALM_EINVAL, "lora_down_drop: null pointer");
  if (!aligned(x, 16) || !aligned(a0, 16) || (two && !aligned(a1, 16)))
    return fail(TALM_EINVAL, "lora_down_drop: x and the A matrices must be 16-byte aligned");
  DownArgs a{};
  a.x = x; a.ldx = ldx; a.n_tokens = static_cast<int>(n_tokens); a.k = static_cast<int>(k);
  a.n_adapters = n_adapters; a.parts = 1;
  a.a[0] = a0; a.a[1] = two ? a1 : a0;
  a.scaling[0] = scaling0; a.scaling[1] = scaling1;
  a.drop = DropArgs{key, 0, drop_threshold(p)};
  a.site[0] = site0; a.site[1] = site1;
  a.factor = drop_factor(a.drop.threshold);
  a.t = t; a.ts = ts; a.ldt = ldt;
  launch_down(a, as_stream(stream));
  return check_launch("lora_down_drop");
}

TALM_API int64_t talm_lora_branch_fwd_workspace(int64_t n_tokens, int64_t k) {
  if (n_tokens < 0 || n_tokens > (1 << 30) || k < 32 || k % 32) return -1;
  return down_parts(n_tokens, k) * n_tokens * kRank * 4;
}

TALM_API int talm_lora_branch_fwd(const uint16_t* x, int64_t ldx, int64_t n_tokens, int64_t k, int64_t cols,
                                  const uint16_t* a_, const uint16_t* b, float p, const int64_t* key,
                                  uint32_t site, float scaling, uint16_t* t, uint16_t* y, void* workspace,
                                  int64_t workspace_bytes, void* stream) {
  const int64_t need = talm_lora_branch_fwd_workspace(n_tokens, k);
  if (need < 0 || n_tokens > kUpTokens * int64_t{65535} || ldx < k || ldx % 8 || cols < 8 || cols % 8 ||
      cols > (1 << 30) || !fits32(16, ldx) || !fits32(16, k))
    return fail(TALM_EINVAL,
                "lora_branch_fwd: bad shape (tokens %lld, k %lld, ldx %lld, columns %lld): k a multiple of 32 "
                "inside x's rows of a multiple of 8, columns a multiple of 8",
                (long long)n_tokens, (long long)k, (long long)ldx, (long long)cols);
  const int status = check_drop("lora_branch_fwd", key, p);
  if (status != TALM_OK) return status;
  if (n_tokens == 0) return ok();
  if (!x || !a_ || !b || !t || !y) return fail(TALM_EINVAL, "lora_branch_fwd: null pointer");
  if (!aligned(x, 16) || !aligned(a_, 16) || !aligned(b, 16) || !aligned(t, 16) || !aligned(y, 16))
    return fail(TALM_EINVAL, "lora_branch_fwd: operands must be 16-byte aligned");
  if (!workspace || workspace_bytes < need || !aligned(workspace, 16))
    return fail(TALM_EINVAL, "lora_branch_fwd: a 16-byte aligned workspace of %lld bytes is needed", (long long)need);
  DownArgs d{};
  d.x = x; d.ldx = ldx; d.n_tokens = static_cast<int>(n_tokens); d.k = static_cast<int>(k);
  d.n_adapters = 1; d.parts = down_parts(n_tokens, k);
  d.a[0] = d.a[1] = a_;
  d.drop = DropArgs{key, 0, drop_threshold(p)};
  d.site[0] = site;
  d.part = static_cast<float*>(workspace);
  const hipStream_t s = as_stream(stream);
  launch_down(d, s);
  UpArgs u{};
  u.part = d.part; u.parts = d.parts; u.n_tokens = d.n_tokens; u.cols = static_cast<int>(cols);
  u.factor = drop_factor(d.drop.threshold); u.scaling = scaling;
  u.t = t; u.b = b; u.y = y;
  hipLaunchKernelGGL(lora_up_kernel,
                     dim3(static_cast<unsigned>((cols + 127) / 128),
                          static_cast<unsigned>((n_tokens + kUpTokens - 1) / kUpTokens)),
                     dim3(256), 0, s, u);
  return check_launch("lora_branch_fwd");
}

TALM_API int64_t talm_lora_bwd_drop_workspace(int64_t n_tokens, int64_t hidden, int32_t n_adapters, int64_t seg0,
                                              int64_t seg1) {
  if (n_tokens < 0 || n_tokens > (1 << 30) || hidden < 8 || hidden % 8 || hidden > (1 << 26) || n_adapters < 1 ||
      n_adapters > kMaxAdapters || seg0 < 8 || seg0 % 8 || seg0 > (1 << 26) ||
      (n_adapters > 1 && (seg1 < 8 || seg1 % 8 || seg1 > (1 << 26))))
    return -1;
  const BwdPlan w = bwd_plan(n_tokens, hidden, n_adapters, seg0, seg1);
  return w.chunks > 65535 ? -1 : w.chunks * w.cols * kRank * 4;
}

TALM_API int talm_lora_bwd_drop(const uint16_t* x, int64_t ldx, const uint16_t* dy, int64_t ldy,
                                const uint16_t* u, int64_t ldu, const uint16_t* t, int64_t ldt,
                                int64_t n_tokens, int64_t hidden, int32_t n_adapters, float p,
                                const int64_t* key, uint32_t site0, uint32_t site1, int32_t grad_dtype,
                                int64_t lo0, int64_t seg0, float scaling0, void* da0, void* db0, int64_t lo1,
                                int64_t seg1, float scaling1, void* da1, void* db1, const uint16_t* a0,
                                const uint16_t* a1, const uint16_t* base, int64_t ldb, uint16_t* dx, int64_t ldd,
                                void* workspace, int64_t workspace_bytes, void* stream) {
  const bool two = n_adapters > 1;
  const int64_t need = talm_lora_bwd_drop_workspace(n_tokens, hidden, n_adapters, seg0, seg1);
  if (need < 0 || ldx < hidden || ldx % 8 || ldy % 8 || lo0 < 0 || lo0 % 8 || lo0 + seg0 > ldy ||
      (two && (lo1 < 0 || lo1 % 8 || lo1 + seg1 > ldy)) || ldu < kRank * n_adapters || ldu % 8 ||
      ldt < kRank * n_adapters || ldt % 8 ||
      (dx && (ldd < hidden || ldd % 8 || (base && (ldb < hidden || ldb % 8)))))
    return fail(TALM_EINVAL,
                "lora_bwd_drop: bad shape (tokens %lld, hidden %lld, segments %lld/%lld at %lld/%lld, strides "
                "%lld/%lld/%lld/%lld, adapters %d): sizes and strides multiples of 8, 1-2 adapters of rank 16",
                (long long)n_tokens, (long long)hidden, (long long)seg0, (long long)seg1, (long long)lo0,
                (long long)lo1, (long long)ldx, (long long)ldy, (long long)ldu, (long long)ldt, n_adapters);
  if (grad_dtype != TALM_F32 && grad_dtype != TALM_F16)
    return fail(TALM_EINVAL, "lora_bwd_drop: gradients of dtype %d", grad_dtype);
  const int status = check_drop("lora_bwd_drop", key, p);
  if (status != TALM_OK) return status;
  const bool grads = da0 != nullptr;
  if (grads ? !db0 || (two && (!da1 || !db1)) : db0 || da1 || db1)
    return fail(TALM_EINVAL, "lora_bwd_drop: the weight gradients are given all or none");
  if (n_tokens == 0) dx = nullptr;  // no element, and A may be null
  if (!grads && !dx) return ok();
  if (n_tokens > 0 && (!x || !dy || !u || !t || (dx && (!a0 || (two && !a1)))))
    return fail(TALM_EINVAL, "lora_bwd_drop: null pointer");
  if (!aligned(x, 16) || !aligned(dy, 16) || !aligned(u, 16) || !aligned(t, 16) || !aligned(base, 16) ||
      !aligned(dx, 16))
    return fail(TALM_EINVAL, "lora_bwd_drop: operands must be 16-byte aligned");
  if (!workspace || workspace_bytes < need || !aligned(workspace, 16))
    return fail(TALM_EINVAL, "lora_bwd_drop: a 16-byte aligned workspace of %lld bytes is needed", (long long)need);
  const BwdPlan w = bwd_plan(n_tokens, hidden, n_adapters, seg0, seg1);
  BwdArgs a{};
  a.x = x; a.ldx = ldx; a.dy = dy; a.ldy = ldy; a.u = u; a.ldu = ldu; a.t = t; a.ldt = ldt;
  a.n_tokens = static_cast<int>(n_tokens); a.hidden = static_cast<int>(hidden); a.n_adapters = n_adapters;
  a.lo[0] = static_cast<int>(lo0); a.lo[1] = static_cast<int>(lo1);
  a.seg[0] = static_cast<int>(seg0); a.seg[1] = static_cast<int>(seg1);
  a.scaling[0] = scaling0; a.scaling[1] = scaling1;
  a.drop = DropArgs{key, 0, drop_threshold(p)};
  a.site[0] = site0; a.site[1] = site1;
  a.factor = drop_factor(a.drop.threshold);
  a.a[0] = a0; a.a[1] = two ? a1 : a0;
  a.base = base; a.ldb = ldb; a.dx = dx; a.ldd = ldd;
  auto pad = [](int64_t n) { return static_cast<int>((n + 127) / 128 * 128); };
  for (int job = 0; job < 2 * n_adapters; ++job)
    a.first[job + 1] = a.first[job] + pad(job < n_adapters ? a.hidden : a.seg[job - n_adapters]);
  a.cols = static_cast<int>(w.cols);
  a.chunk = static_cast<int>(w.chunk); a.chunks = static_cast<int>(w.chunks);
  a.part = static_cast<float*>(workspace);
  a.half_out = grad_dtype == TALM_F16;
  a.da[0] = da0; a.da[1] = da1; a.db[0] = db0; a.db[1] = db1;
  const hipStream_t s = as_stream(stream);
  const int64_t blocks = w.cols / 128 - (n_adapters - 1) * w.x_blocks;  // x's blocks serve every adapter
  const dim3 grid(static_cast<unsigned>(grads ? blocks : w.x_blocks), static_cast<unsigned>(w.chunks));
  if (two) hipLaunchKernelGGL(lora_bwd_drop_kernel<2>, grid, dim3(256), 0, s, a);
  else hipLaunchKernelGGL(lora_bwd_drop_kernel<1>, grid, dim3(256), 0, s, a);
  if (grads)
    hipLaunchKernelGGL(lora_wgrad_sum_kernel, dim3(static_cast<unsigned>((w.cols * kRank + 255) / 256)), dim3(256), 0,
                       s, a);
  return check_launch("lora_bwd_drop");
}
