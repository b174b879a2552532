// Products of a few tokens (1 .. 32) with a weight W [rows, cols] held in the layer group's NF4 form,
// for the calls that answer token by token: out = x W^T + bias (+ LoRA adapters, ts B^T). Every weight is read once as its
// 4-bit code, with its block's absmax code and second-level scale, and never written out; the fp16
// weights are bit-identical to talm_nf4_group_dequant's (solution/qgroup.py:72-99), the products fp32.
//
// The weights are the A operand of v_mfma_f32_16x16x32_f16, the tokens the B operand. A lane takes
// whole 64-weight blocks (32 contiguous bytes of codes, one scale) and looks their weights up in a
// table of the block's 16 scaled levels kept in its registers (nf4_code.h); the reduction's order is
// free, so eight MFMAs take a block's eight-weight words as they lie, against the same columns of x.
// Sixteen operand rows are 16 / P rows of W times P parts of the reduction (unit: 256 P columns); the
// operand's columns are the tokens times the same P parts, and the blocks of the result where both
// parts agree are summed: few tokens leave operand columns free, and small P tiles give short rows
// of W enough workgroups. The wavefronts of a workgroup split the units, joined through LDS in order.
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
};

constexpr int kGemvMaxWaves = 16;
constexpr int kGemvTokens = 32;

template <int P, int TB>
__global__ __launch_bounds__(64 * kGemvMaxWaves) void nf4_gemv_rows_kernel(GemvArgs a) {
  static_assert(TB == 1 || P == 1, "two token blocks need every operand column");
  constexpr int R = 16 / P;  // rows of W, and tokens per block
  __shared__ float table[256];
  __shared__ float red[kGemvMaxWaves][TB][P][R][R + 1];
  const int tid = threadIdx.x, lane = tid & 63, waves = blockDim.x >> 6;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int m = lane & 15, g = lane >> 4;
  const int row0 = blockIdx.x * R;
  const int wr = m % R, part = m / R;  // this lane's row of W and part (A); its token and part (B)
  for (int i = tid; i < 256; i += blockDim.x) table[i] = a.code[i];
  __syncthreads();
  const bool row_in = row0 + wr < a.rows;
  const int64_t tile0 = static_cast<int64_t>(row0) * a.cols;  // the tile's first weight
  const __amdgpu_buffer_rsrc_t rw = __builtin_amdgcn_make_buffer_rsrc(
      const_cast<uint8_t*>(a.packed + tile0 / 2), 0, 0x7fffffff, 0x00020000);
  const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc(
      const_cast<uint8_t*>(a.absmax8 + tile0 / 64), 0, 0x7fffffff, 0x00020000);
  const __amdgpu_buffer_rsrc_t rx = buffer_rsrc(a.x);
  f32x4 acc[TB];
#pragma unroll
  for (int b = 0; b < TB; ++b) acc[b] = f32x4{0.f, 0.f, 0.f, 0.f};
  for (int u = wave; u < a.units; u += waves) {
    const int k = (u * P + part) * 256 + 64 * g;
    const bool k_in = k < a.cols, in = k_in && row_in;
    const uint32_t e = static_cast<uint32_t>(wr * a.cols + k);  // weight index inside the tile
    const uint4 w0 = __builtin_bit_cast(uint4, __builtin_amdgcn_raw_buffer_load_b128(rw, in ? e / 2 : kOob, 0, 0));
    const uint4 w1 =
        __builtin_bit_cast(uint4, __builtin_amdgcn_raw_buffer_load_b128(rw, in ? e / 2 + 16 : kOob, 0, 0));
    const uint8_t a8 = __builtin_amdgcn_raw_buffer_load_b8(rs, in ? e / 64 : kOob, 0, 0);
    const int64_t i2 = in ? ((tile0 + e) >> 6) >> a.shift2 : 0;
    const float s2 = a.absmax2[i2], o2 = a.offset2[i2];
    uint4 xv[TB][8];
#pragma unroll
    for (int b = 0; b < TB; ++b) {
      const int tok = wr + R * b;
      const uint32_t off = k_in && tok < a.M ? static_cast<uint32_t>((tok * a.ldx + k) * 2) : kOob;
#pragma unroll
      for (int j = 0; j < 8; ++j)
        xv[b][j] = __builtin_bit_cast(uint4, __builtin_amdgcn_raw_buffer_load_b128(rx, off, 16 * j, 0));
    }
    const float scale = in ? block_scale(table[a8], s2, o2) : 0.f;
    const Nf4Table t = nf4_table(scale);
    const uint32_t words[8] = {w0.x, w0.y, w0.z, w0.w, w1.x, w1.y, w1.z, w1.w};
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const half8_t wf = __builtin_bit_cast(half8_t, nf4_lookup_word(words[j], t));
#pragma unroll
      for (int b = 0; b < TB; ++b)
        acc[b] = __builtin_amdgcn_mfma_f32_16x16x32_f16(wf, __builtin_bit_cast(half8_t, xv[b][j]), acc[b], 0, 0, 0);
    }
  }
  // element v of lane l: operand row 4 (l / 16) + v, column l % 16
#pragma unroll
  for (int b = 0; b < TB; ++b)
#pragma unroll
    for (int v = 0; v < 4; ++v) {
      const int r = 4 * g + v;
      if (r / R == part) red[wave][b][part][r % R][wr] = acc[b][v];
    }
  __syncthreads();
  for (int i = tid; i < TB * R * R; i += blockDim.x) {
    const int r = i % R, tok = i / R % R, b = i / (R * R), row = row0 + r;
    if (row >= a.rows || tok + R * b >= a.M) continue;
    float sum = 0.f;
    for (int w = 0; w < waves; ++w)
#pragma unroll
      for (int p = 0; p < P; ++p) sum += red[w][b][p][r][tok];
    if (a.bias) sum += h2f(a.bias[row]);
    if (a.ts) {
#pragma unroll
      for (int ad = 0; ad < 2; ++ad)
        if (row >= a.lo[ad] && row < a.hi[ad]) {
          const uint16_t* tp = a.ts + static_cast<int64_t>(tok + R * b) * a.ldt + 16 * ad;
          const uint16_t* bp = a.b[ad] + static_cast<int64_t>(row - a.lo[ad]) * 16;
#pragma unroll
          for (int q = 0; q < 16; ++q) sum += h2f(tp[q]) * h2f(bp[q]);
        }
    }
    a.out[static_cast<int64_t>(tok + R * b) * a.ldo + row] = f2h(sum);
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
      cols > (1 << 26) || ldx < cols || ldx % 8 || ldx > (1 << 24) || ldo < rows)
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
  // parts of the reduction per tile: what the tokens leave room for, fewest idle lanes and CUs
  int best = 1;
  double cost = 0;
  for (int p = 1; p <= 4 && p * n_tokens <= 16; p *= 2) {
    const int64_t units = (cols + 256 * p - 1) / (256 * p), wgs = (rows * p + 15) / 16;
    const double waste = static_cast<double>(units * 256 * p) / cols, cus = device_cus();
    const double c = waste * std::max(1.0, cus / static_cast<double>(wgs));
    if (cost == 0 || c < cost) { cost = c; best = p; }
  }
  a.units = static_cast<int>((cols + 256 * best - 1) / (256 * best));
  const int turns = (a.units + kGemvMaxWaves - 1) / kGemvMaxWaves, waves = (a.units + turns - 1) / turns;
  const dim3 grid(static_cast<unsigned>((rows * best + 15) / 16)), block(64 * waves);
  const hipStream_t s = as_stream(stream);
  if (n_tokens > 16) hipLaunchKernelGGL((nf4_gemv_rows_kernel<1, 2>), grid, block, 0, s, a);
  else if (best == 1) hipLaunchKernelGGL((nf4_gemv_rows_kernel<1, 1>), grid, block, 0, s, a);
  else if (best == 2) hipLaunchKernelGGL((nf4_gemv_rows_kernel<2, 1>), grid, block, 0, s, a);
  else hipLaunchKernelGGL((nf4_gemv_rows_kernel<4, 1>), grid, block, 0, s, a);
  return check_launch("nf4_gemv");
}
