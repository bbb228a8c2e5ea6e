// Quantizer to 8-bit floating point with a scale for each block of 128 (gfx950), and its inverse.
//
// A workgroup of 256 threads takes 128 rows x 128 columns, so that every block of either copy (1 x 128, 128 x 1, 128 x 128) lies in one workgroup and x is
// read once, whatever is made of it.  A thread holds 8 rows x 8 columns in registers: 16 threads across a row (256 bytes of bf16), and the codes of
// 8 tokens of a column are 8 bytes of the transposed copy.  Those go through the LDS, so that both copies leave as whole 128-byte lines.
//
// code = RNE(x L / amax) is meant exactly.  With L = 0.875 2^k:  t = 0.875 x  and  a = amax 2^-k  (no overflow, and for bf16 data both are exact), r = RN(1 / a),
//   q = t r,   e = q a - t,   q - e r
// is t / a rounded correctly (Markstein), so a quotient of bf16 numbers that lies halfway between two codes is that midpoint in fp32 too and
// goes to the even code; q alone is a rounding off, and one code in 300 of Gaussian bf16 data was the other neighbour.  Of fp32 data t and the quotient are rounded to fp32
// ahead of the code: one within 2^-22 of a midpoint may take the other neighbour.
//
// What bounds it is HBM: 4096 x 14336 of a weight, both copies, 49.6 us in a stream of such calls (4.7 TB/s; 38 us, 6.2 TB/s, where x is still cached), 32 experts of 5760 x 2880 411 us
// (5.2 TB/s, what a large copy reaches); 8192 x 4096 of activations, both copies, 28.8.  Below 2000 tiles all loads, then all stores, are under way at once and
// their latencies add up: 2048 x 4096 12.8 us, one row 3.6.
#include "fp8.h"

namespace alto {
namespace {

struct Fp8QuantArgs {
  const void* x;
  uint8_t *row_codes, *col_codes;
  float *row_scales, *col_scales;
  const int32_t* offs;
  int64_t M, C, x_sb, x_sm, row_sb, row_ld, col_sb, col_ld;
  int64_t tiles_m, tiles_c, blocks_m;   // tiles along M of this launch (token blocks by groups) and C; blocks of scales along M
  int groups;
};

__device__ __forceinline__ uint32_t umax(uint32_t a, uint32_t b) { return a > b ? a : b; }
// largest of each of the two 16-bit halves
__device__ __forceinline__ uint32_t umax2(uint32_t a, uint32_t b) {
  typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
  return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(u16x2, a), __builtin_bit_cast(u16x2, b)));
}

// What a block's codes need of its amax (bits of the magnitude: NaN is above infinity there): a and 1/a as above; the scale.
struct BlockScale {
  float a, r, scale;
};
template <int CODE>
__device__ __forceinline__ BlockScale block_scale(uint32_t amax_bits) {
  constexpr float FLOOR = Fp8<CODE>::LARGEST * 0x1p-100f;
  const uint32_t bits = umax(amax_bits, __builtin_bit_cast(uint32_t, FLOOR));
  const float amax = u2f(bits);
  const float a = amax * (1.0f / Fp8<CODE>::TWO_K);
  return {a, 1.0f / a, amax / Fp8<CODE>::LARGEST};
}
__device__ __forceinline__ float code_quotient(float t, float a, float r) {
  const float q = t * r;
  return __builtin_fmaf(-__builtin_fmaf(q, a, -t), r, q);   // (the signs this way round keep a -0)
}

// 8 elements of a row as fp32 from bf16 pairs or as they are
template <typename T>
struct Octet;
template <>
struct Octet<__bf16> {
  uint32_t w[4];
  __device__ __forceinline__ float at(int j) const { return j & 1 ? bf16_hi(w[j / 2]) : bf16_lo(w[j / 2]); }
};
template <>
struct Octet<float> {
  uint32_t w[8];
  __device__ __forceinline__ float at(int j) const { return u2f(w[j]); }
};

// VEC: x's rows start at multiples of 16 bytes, and so do the pieces of 8 columns
template <typename T, bool VEC>
__device__ __forceinline__ Octet<T> load_octet(const T* p, int64_t n) {   // n: columns of the piece that exist
  Octet<T> o;
  constexpr int WORDS = sizeof(o.w) / 4;
  if (VEC && n >= 8) {
    const uint4 v = *reinterpret_cast<const uint4*>(p);
    o.w[0] = v.x; o.w[1] = v.y; o.w[2] = v.z; o.w[3] = v.w;
    if constexpr (WORDS == 8) {
      const uint4 u = *reinterpret_cast<const uint4*>(p + 4);
      o.w[4] = u.x; o.w[5] = u.y; o.w[6] = u.z; o.w[7] = u.w;
    }
    return o;
  }
#pragma unroll
  for (int i = 0; i < WORDS; ++i) o.w[i] = 0;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    if (j >= n) continue;
    if constexpr (WORDS == 8) o.w[j] = reinterpret_cast<const uint32_t*>(p)[j];
    else o.w[j / 2] |= (uint32_t) reinterpret_cast<const uint16_t*>(p)[j] << (16 * (j & 1));
  }
  return o;
}

// OUT: 1 row copy, 2 col copy, 3 both
template <typename T, int CODE, int OUT, bool B2D, bool VEC>
__global__ __launch_bounds__(256) void fp8_quantize_kernel(const Fp8QuantArgs p) {
  constexpr bool ROW = OUT & 1, COL = OUT & 2;
  __shared__ __attribute__((aligned(16))) uint8_t turned[COL ? 128 * 128 : 16];
  __shared__ uint32_t row_amax[128], col_amax[4][128];
  __shared__ float2 row_ar[128], col_ar[128];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, l16 = tid & 15, rg = tid >> 4;
  // consecutive workgroups: the tiles of a band of rows
  const int64_t tile_c = blockIdx.x % p.tiles_c, tile_m = blockIdx.x / p.tiles_c % p.tiles_m, batch = blockIdx.x / p.tiles_c / p.tiles_m;
  int64_t m0 = tile_m * 128, m1 = m0 + 128 < p.M ? m0 + 128 : p.M;
  if (p.offs != nullptr) {
    const Segment s = find_piece(p.offs, p.groups, p.M, 128, tile_m);
    m0 = s.lo;
    m1 = s.hi;
  }
  const int rows = (int)(m1 - m0);   // 0 .. 128
  const int64_t c0 = tile_c * 128 + 8 * l16, cols = p.C - c0;   // this thread's 8 columns; how many of them (and behind them) exist
  const T* x = reinterpret_cast<const T*>(p.x) + batch * p.x_sb + m0 * p.x_sm + c0;

  Octet<T> v[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int m = 8 * rg + i;
    if (m < rows && cols > 0) v[i] = load_octet<T, VEC>(x + m * p.x_sm, cols);
    else v[i] = Octet<T>{};
  }

  // ---- amax: rows across 16 lanes, columns across the 8 rows here, 4 groups of rows of the wave and 4 waves
  uint32_t cmax[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) cmax[j] = 0;
  if constexpr (sizeof(T) == 2) {
    uint32_t c2[4] = {0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      uint32_t r2 = 0;
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const uint32_t m = v[i].w[w] & 0x7FFF7FFFu;
        r2 = umax2(r2, m);
        c2[w] = umax2(c2[w], m);
      }
      uint32_t r = umax(r2 & 0xFFFFu, r2 >> 16);
      r = umax(r, dpp_u32<ALTO_DPP_QUAD_XOR1>(r));
      r = umax(r, dpp_u32<ALTO_DPP_QUAD_XOR2>(r));
      r = umax(r, dpp_u32<ALTO_DPP_HALF_MIRROR>(r));
      r = umax(r, dpp_u32<ALTO_DPP_ROW_ROR8>(r));
      if (l16 == 0) row_amax[8 * rg + i] = r << 16;
    }
    if constexpr (COL || B2D) {
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        c2[w] = umax2(c2[w], __shfl_xor(c2[w], 16));
        c2[w] = umax2(c2[w], __shfl_xor(c2[w], 32));
        cmax[2 * w] = c2[w] << 16;
        cmax[2 * w + 1] = c2[w] & 0xFFFF0000u;
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      uint32_t r = 0;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const uint32_t m = v[i].w[j] & 0x7FFFFFFFu;
        r = umax(r, m);
        cmax[j] = umax(cmax[j], m);
      }
      r = umax(r, dpp_u32<ALTO_DPP_QUAD_XOR1>(r));
      r = umax(r, dpp_u32<ALTO_DPP_QUAD_XOR2>(r));
      r = umax(r, dpp_u32<ALTO_DPP_HALF_MIRROR>(r));
      r = umax(r, dpp_u32<ALTO_DPP_ROW_ROR8>(r));
      if (l16 == 0) row_amax[8 * rg + i] = r;
    }
    if constexpr (COL || B2D) {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        cmax[j] = umax(cmax[j], __shfl_xor(cmax[j], 16));
        cmax[j] = umax(cmax[j], __shfl_xor(cmax[j], 32));
      }
    }
  }
  if constexpr (COL || B2D) {
    if (lane < 16) {
#pragma unroll
      for (int j = 0; j < 8; ++j) col_amax[wave][8 * l16 + j] = cmax[j];
    }
  }
  __syncthreads();

  // ---- scales: one thread a row, one a column; blocks of 128 x 128: every wave the whole block's
  float block_a = 0, block_r = 0;
  if constexpr (B2D) {
    uint32_t m = umax(row_amax[lane], row_amax[lane + 64]);
#pragma unroll
    for (int d = 1; d < 64; d *= 2) m = umax(m, __shfl_xor(m, d));
    const BlockScale s = block_scale<CODE>(m);
    block_a = s.a;
    block_r = s.r;
    if (tid == 0) p.row_scales[(batch * p.blocks_m + tile_m) * p.tiles_c + tile_c] = s.scale;
  } else {
    if (ROW && tid < 128) {
      const BlockScale s = block_scale<CODE>(row_amax[tid]);
      row_ar[tid] = make_float2(s.a, s.r);
      if (tid < rows) p.row_scales[(batch * p.tiles_c + tile_c) * p.M + m0 + tid] = s.scale;
    }
    if (COL && tid >= 128) {
      const int c = tid - 128;
      const BlockScale s = block_scale<CODE>(umax(umax(col_amax[0][c], col_amax[1][c]), umax(col_amax[2][c], col_amax[3][c])));
      col_ar[c] = make_float2(s.a, s.r);
      if (tile_c * 128 + c < p.C) p.col_scales[(batch * p.blocks_m + tile_m) * p.C + tile_c * 128 + c] = s.scale;
    }
    __syncthreads();
  }

  // ---- codes
  constexpr bool SAME = B2D;   // both copies hold the same codes
  const int64_t c16 = (p.C + 15) / 16 * 16;   // columns of a row of codes that are written
  float2 car[8];
  if constexpr (COL && !SAME) {
#pragma unroll
    for (int j = 0; j < 8; ++j) car[j] = col_ar[8 * l16 + j];
  }
  int cw[8][2];   // of each of the 8 columns: the codes of the 8 rows
#pragma unroll
  for (int j = 0; j < 8; ++j) cw[j][0] = cw[j][1] = 0;
#pragma unroll
  for (int i = 0; i < 8; i += 2) {   // two rows at a time: two tokens of a column are half a dword
    float qc[2][8];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int m = 8 * rg + i + h;
      float a = block_a, r = block_r;
      if constexpr (ROW && !SAME) {
        const float2 ar = row_ar[m];
        a = ar.x;
        r = ar.y;
      }
      float q[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float t = 0.875f * v[i + h].at(j);
        if constexpr (ROW || SAME) q[j] = code_quotient(t, a, r);
        if constexpr (COL) qc[h][j] = SAME ? q[j] : code_quotient(t, car[j].x, car[j].y);
      }
      if constexpr (ROW) {
        int w0 = Fp8<CODE>::template pack<false>(q[0], q[1], 0), w1 = Fp8<CODE>::template pack<false>(q[4], q[5], 0);
        w0 = Fp8<CODE>::template pack<true>(q[2], q[3], w0);
        w1 = Fp8<CODE>::template pack<true>(q[6], q[7], w1);
        // (columns at or beyond C hold zeros: with a NaN scale their codes would not)
        if (cols < 8) {
          const uint64_t keep = cols <= 0 ? 0ull : (1ull << (8 * cols)) - 1ull;
          w0 &= (int)keep;
          w1 &= (int)(keep >> 32);
        }
        if (m < rows && c0 < c16) *reinterpret_cast<int2*>(p.row_codes + batch * p.row_sb + (m0 + m) * p.row_ld + c0) = make_int2(w0, w1);
      }
    }
    if constexpr (COL) {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        cw[j][i / 4] = i % 4 == 0 ? Fp8<CODE>::template pack<false>(qc[0][j], qc[1][j], cw[j][i / 4]) : Fp8<CODE>::template pack<true>(qc[0][j], qc[1][j], cw[j][i / 4]);
    }
  }
  if constexpr (COL) {
    // column c's 128 tokens: 16 slots of 8 bytes, slot g of rows 8 g .. at place g ^ (c / 8) % 16
    const int valid = rows - 8 * rg;   // tokens of this thread that exist; the others hold zeros
    const uint64_t keep = valid <= 0 ? 0ull : valid >= 8 ? ~0ull : (1ull << (8 * valid)) - 1ull;
#pragma unroll
    for (int j = 0; j < 8; ++j)
      *reinterpret_cast<int2*>(turned + (8 * l16 + j) * 128 + 8 * (rg ^ l16)) = make_int2(cw[j][0] & (int)keep, cw[j][1] & (int)(keep >> 32));
    __syncthreads();
    const int64_t t0 = tile_m * 128;                                      // place of the tile's tokens in the rows of codes
    const int64_t t16 = p.offs != nullptr ? t0 + 128 : (p.M + 15) / 16 * 16;   // written up to there
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int piece = 256 * k + tid, c = piece / 8, s = piece % 8, turn = (c / 8) & 15;   // 16 bytes: slots 2 s, 2 s + 1
      int4 w = *reinterpret_cast<const int4*>(turned + c * 128 + 16 * (s ^ (turn >> 1)));
      if (turn & 1) w = make_int4(w.z, w.w, w.x, w.y);
      if (tile_c * 128 + c < p.C && t0 + 16 * s < t16) *reinterpret_cast<int4*>(p.col_codes + batch * p.col_sb + (tile_c * 128 + c) * p.col_ld + t0 + 16 * s) = w;
    }
  }
}

template <typename T, int CODE, int OUT, bool B2D>
void launch_vec(const Fp8QuantArgs& a, bool vec, dim3 grid, hipStream_t st) {
  if (vec) hipLaunchKernelGGL((fp8_quantize_kernel<T, CODE, OUT, B2D, true>), grid, dim3(256), 0, st, a);
  else hipLaunchKernelGGL((fp8_quantize_kernel<T, CODE, OUT, B2D, false>), grid, dim3(256), 0, st, a);
}
template <typename T, int CODE>
void launch_quantize(const Fp8QuantArgs& a, int out, bool is_2d, bool vec, dim3 grid, hipStream_t st) {
  if (is_2d) {
    if (out == 1) launch_vec<T, CODE, 1, true>(a, vec, grid, st);
    else if (out == 2) launch_vec<T, CODE, 2, true>(a, vec, grid, st);
    else launch_vec<T, CODE, 3, true>(a, vec, grid, st);
  } else {
    if (out == 1) launch_vec<T, CODE, 1, false>(a, vec, grid, st);
    else if (out == 2) launch_vec<T, CODE, 2, false>(a, vec, grid, st);
    else launch_vec<T, CODE, 3, false>(a, vec, grid, st);
  }
}

bool valid_stride(int64_t s) { return s >= 0 && s < (1ll << 40); }

}  // namespace

static int fp8_quantize(const alto_mxfp4_fp8_quantize_t& p, hipStream_t st) {
  ALTO_REQUIRE(p.dtype == ALTO_DT_BF16 || p.dtype == ALTO_DT_F32, "fp8_quantize: dtype %d is neither bf16 (0) nor f32 (1)", p.dtype);
  ALTO_REQUIRE(p.code == ALTO_FP8_E4M3 || p.code == ALTO_FP8_E5M2, "fp8_quantize: code %d is neither E4M3 (0) nor E5M2 (1)", p.code);
  ALTO_REQUIRE(p.B >= 0 && p.M >= 0 && p.C >= 0 && p.M < (1ll << 31) && p.C < (1ll << 31), "fp8_quantize: size out of range");
  ALTO_REQUIRE(p.row_codes || p.col_codes, "fp8_quantize: no output");
  ALTO_REQUIRE(!p.offs || (p.B == 1 && p.col_codes && !p.is_2d && p.groups >= 1 && p.groups < (1 << 20)), "fp8_quantize: groups need B = 1, a col copy, blocks along the rows");
  if (p.B == 0 || p.C == 0 || (p.M == 0 && !p.offs)) return ALTO_MXFP4_OK;
  const int64_t size = p.dtype == ALTO_DT_BF16 ? 2 : 4;
  ALTO_REQUIRE(p.x || p.M == 0, "fp8_quantize: null pointer");
  ALTO_REQUIRE(p.is_2d ? p.row_scales != nullptr : (!p.row_codes || p.row_scales) && (!p.col_codes || p.col_scales), "fp8_quantize: null scales");
  ALTO_REQUIRE((uintptr_t)p.x % (uintptr_t)size == 0 && ((uintptr_t)p.row_codes | (uintptr_t)p.col_codes) % 16 == 0 && ((uintptr_t)p.row_scales | (uintptr_t)p.col_scales | (uintptr_t)p.offs) % 4 == 0,
               "fp8_quantize: misaligned pointer");
  ALTO_REQUIRE(valid_stride(p.x_sb) && valid_stride(p.x_sm) && valid_stride(p.row_sb) && valid_stride(p.row_ld) && valid_stride(p.col_sb) && valid_stride(p.col_ld),
               "fp8_quantize: strides must be non-negative");
  Fp8QuantArgs a{};
  a.tiles_c = (p.C + 127) / 128;
  a.tiles_m = p.offs ? most_pieces(p.M, p.groups, 128) : (p.M + 127) / 128;
  a.blocks_m = a.tiles_m;
  ALTO_REQUIRE(!p.row_codes || (p.row_ld % 16 == 0 && p.row_sb % 16 == 0 && (p.M <= 1 || p.row_ld >= (p.C + 15) / 16 * 16)), "fp8_quantize: rows of codes overlap or are misaligned");
  const int64_t tokens = p.offs ? a.tiles_m * 128 : (p.M + 15) / 16 * 16;
  ALTO_REQUIRE(!p.col_codes || (p.col_ld % 16 == 0 && p.col_sb % 16 == 0 && (p.C <= 1 || p.col_ld >= tokens)), "fp8_quantize: columns of codes overlap or are misaligned");
  ALTO_REQUIRE(product_below(1ll << 24, a.tiles_c, a.tiles_m, p.B), "fp8_quantize: too many tiles for one launch");   // (its threads, 256 a workgroup, are counted in 32 bits)
  if (a.tiles_m == 0) return ALTO_MXFP4_OK;
  a.x = p.x; a.row_codes = (uint8_t*)p.row_codes; a.col_codes = (uint8_t*)p.col_codes; a.row_scales = p.row_scales; a.col_scales = p.col_scales; a.offs = p.offs;
  a.M = p.M; a.C = p.C; a.x_sb = p.x_sb; a.x_sm = p.x_sm; a.row_sb = p.row_sb; a.row_ld = p.row_ld; a.col_sb = p.col_sb; a.col_ld = p.col_ld; a.groups = p.groups;
  const int64_t unit = 16 / size;
  const bool vec = (uintptr_t)p.x % 16 == 0 && (p.M <= 1 || p.x_sm % unit == 0) && (p.B == 1 || p.x_sb % unit == 0);
  const dim3 grid((unsigned)(a.tiles_c * a.tiles_m * p.B));
  const int out = (p.row_codes ? 1 : 0) | (p.col_codes ? 2 : 0);
  if (p.dtype == ALTO_DT_BF16) {
    if (p.code == ALTO_FP8_E4M3) launch_quantize<__bf16, ALTO_FP8_E4M3>(a, out, p.is_2d, vec, grid, st);
    else launch_quantize<__bf16, ALTO_FP8_E5M2>(a, out, p.is_2d, vec, grid, st);
  } else {
    if (p.code == ALTO_FP8_E4M3) launch_quantize<float, ALTO_FP8_E4M3>(a, out, p.is_2d, vec, grid, st);
    else launch_quantize<float, ALTO_FP8_E5M2>(a, out, p.is_2d, vec, grid, st);
  }
  return check_launch("fp8_quantize");
}

namespace {

struct Fp8DequantArgs {
  const uint8_t* codes;
  const float* scales;
  void* out;
  int64_t R, C, pieces, codes_sb, ld, s_sb, s_r, s_c, out_sb, ldo;
  int shift;   // of the row: 7 with blocks of 128 x 128
};

// 8 codes of a row to a thread; VEC: they and their results are accessed whole
template <typename T, int CODE, bool VEC>
__global__ __launch_bounds__(256) void fp8_dequantize_kernel(const Fp8DequantArgs p) {
  const int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t c0 = at % p.pieces * 8, r = at / p.pieces, batch = blockIdx.y;
  if (r >= p.R) return;
  const uint8_t* q = p.codes + batch * p.codes_sb + r * p.ld + c0;
  const float s = p.scales[batch * p.s_sb + (r >> p.shift) * p.s_r + c0 / 128 * p.s_c];
  T* o = reinterpret_cast<T*>(p.out) + batch * p.out_sb + r * p.ldo + c0;
  const int n = p.C - c0 < 8 ? (int)(p.C - c0) : 8;
  int w[2] = {0, 0};
  if (VEC && n == 8) {
    const int2 v = *reinterpret_cast<const int2*>(q);
    w[0] = v.x; w[1] = v.y;
  } else {
    for (int j = 0; j < n; ++j) w[j / 4] |= (int)q[j] << (8 * (j & 3));
  }
  float f[8] = {Fp8<CODE>::template value<0>(w[0]) * s, Fp8<CODE>::template value<1>(w[0]) * s, Fp8<CODE>::template value<2>(w[0]) * s, Fp8<CODE>::template value<3>(w[0]) * s,
                Fp8<CODE>::template value<0>(w[1]) * s, Fp8<CODE>::template value<1>(w[1]) * s, Fp8<CODE>::template value<2>(w[1]) * s, Fp8<CODE>::template value<3>(w[1]) * s};
  if (VEC && n == 8) {
    if constexpr (sizeof(T) == 2) {
      *reinterpret_cast<uint4*>(o) = make_uint4(pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]), pack_bf16x2(f[4], f[5]), pack_bf16x2(f[6], f[7]));
    } else {
      *reinterpret_cast<float4*>(o) = make_float4(f[0], f[1], f[2], f[3]);
      *reinterpret_cast<float4*>(o + 4) = make_float4(f[4], f[5], f[6], f[7]);
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (j < n) o[j] = (T)f[j];
  }
}

template <typename T, int CODE>
void launch_dequantize(const Fp8DequantArgs& a, bool vec, dim3 grid, hipStream_t st) {
  if (vec) hipLaunchKernelGGL((fp8_dequantize_kernel<T, CODE, true>), grid, dim3(256), 0, st, a);
  else hipLaunchKernelGGL((fp8_dequantize_kernel<T, CODE, false>), grid, dim3(256), 0, st, a);
}

}  // namespace

static int fp8_dequantize(const alto_mxfp4_fp8_dequantize_t& p, hipStream_t st) {
  ALTO_REQUIRE(p.out_dtype == ALTO_DT_BF16 || p.out_dtype == ALTO_DT_F32, "fp8_dequantize: dtype %d is neither bf16 (0) nor f32 (1)", p.out_dtype);
  ALTO_REQUIRE(p.code == ALTO_FP8_E4M3 || p.code == ALTO_FP8_E5M2, "fp8_dequantize: code %d is neither E4M3 (0) nor E5M2 (1)", p.code);
  ALTO_REQUIRE(p.B >= 0 && p.B < 65536 && p.R >= 0 && p.C >= 0 && p.R < (1ll << 31) && p.C < (1ll << 31), "fp8_dequantize: size out of range");
  if (p.B == 0 || p.R == 0 || p.C == 0) return ALTO_MXFP4_OK;
  ALTO_REQUIRE(p.codes && p.scales && p.out, "fp8_dequantize: null pointer");
  const int64_t size = p.out_dtype == ALTO_DT_BF16 ? 2 : 4;
  ALTO_REQUIRE((uintptr_t)p.scales % 4 == 0 && (uintptr_t)p.out % (uintptr_t)size == 0, "fp8_dequantize: misaligned pointer");
  for (const int64_t s : {p.codes_sb, p.ld, p.s_sb, p.s_r, p.s_c, p.out_sb, p.ldo}) ALTO_REQUIRE(valid_stride(s), "fp8_dequantize: strides must be non-negative");
  Fp8DequantArgs a{(const uint8_t*)p.codes, p.scales, p.out, p.R, p.C, (p.C + 7) / 8, p.codes_sb, p.ld, p.s_sb, p.s_r, p.s_c, p.out_sb, p.ldo, p.is_2d ? 7 : 0};
  ALTO_REQUIRE(product_below((1ll << 32) - 256, a.pieces, p.R), "fp8_dequantize: too many elements for one launch");   // (its threads are counted in 32 bits)
  const int64_t groups = (a.pieces * p.R + 255) / 256;
  const bool vec = (uintptr_t)p.codes % 8 == 0 && p.ld % 8 == 0 && p.codes_sb % 8 == 0 && (uintptr_t)p.out % 16 == 0 && p.ldo * size % 16 == 0 && p.out_sb * size % 16 == 0;
  const dim3 grid((unsigned)groups, (unsigned)p.B);
  if (p.out_dtype == ALTO_DT_BF16) {
    if (p.code == ALTO_FP8_E4M3) launch_dequantize<__bf16, ALTO_FP8_E4M3>(a, vec, grid, st);
    else launch_dequantize<__bf16, ALTO_FP8_E5M2>(a, vec, grid, st);
  } else {
    if (p.code == ALTO_FP8_E4M3) launch_dequantize<float, ALTO_FP8_E4M3>(a, vec, grid, st);
    else launch_dequantize<float, ALTO_FP8_E5M2>(a, vec, grid, st);
  }
  return check_launch("fp8_dequantize");
}

}  // namespace alto

extern "C" int64_t alto_mxfp4_fp8_token_blocks(int64_t M, int64_t groups) {
  if (M < 0 || groups < 0 || M >= (1ll << 31) || groups >= (1 << 20)) return -1;
  return alto::most_pieces(M, groups, 128);
}
extern "C" int alto_mxfp4_fp8_quantize(const alto_mxfp4_fp8_quantize_t* p, void* stream) {
  ALTO_REQUIRE(p, "fp8_quantize: null pointer");
  return alto::fp8_quantize(*p, (hipStream_t)stream);
}
extern "C" int alto_mxfp4_fp8_dequantize(const alto_mxfp4_fp8_dequantize_t* p, void* stream) {
  ALTO_REQUIRE(p, "fp8_dequantize: null pointer");
  return alto::fp8_dequantize(*p, (hipStream_t)stream);
}
