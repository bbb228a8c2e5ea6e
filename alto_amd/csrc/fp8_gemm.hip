// Products of 8-bit floating-point operands with a scale for each block of 128 (fp8_tile.h): one weight.
#include <utility>

#include "fp8_rows.h"
#include "fp8_tile.h"

namespace alto {
namespace {

typedef Fp8Tile<2, 4, 8> Large;   // 256 x 256, one workgroup a compute unit
typedef Fp8Tile<2, 2, 4> Small;   // 128 x 128, two of them
typedef Fp8Tile<2, 2, 4, 2> Split;   // 128 x 128, one of them, each half of its waves takes half of K
typedef Fp8Tile<1, 1, 4, 4> Four;    // 64 x 64, one of them, each of its 4 waves takes a quarter of K

struct Fp8GemmArgs {
  const uint8_t *a, *b;
  const float *a_scales, *b_scales;
  void* c;
  int64_t M, N, K, lda, ldb, a_ss_r, a_ss_k, b_ss_r, b_ss_k, ldc;
  int a_shift, b_shift, tiles_m, tiles_n, whole, vec;   // whole: tiles of an XCD that stay whole
};

template <class W, int CODE_A, bool B1D, typename OutT>
__device__ __forceinline__ void product(const Fp8GemmArgs& p, int64_t m0, int64_t n0, uint8_t* smem) {
  Fp8TileArgs t;
  t.A = {p.a + m0 * p.lda, p.a_scales + (m0 >> p.a_shift) * p.a_ss_r, p.lda, p.a_ss_r, p.a_ss_k, (int)(p.M - m0 < W::TM ? p.M - m0 : W::TM), p.a_shift};
  t.B = {p.b + n0 * p.ldb, p.b_scales + (n0 >> p.b_shift) * p.b_ss_r, p.ldb, p.b_ss_r, p.b_ss_k, (int)(p.N - n0 < W::TN ? p.N - n0 : W::TN), p.b_shift};
  t.K = p.K;
  fp8_tile_product<W, CODE_A, B1D>(t, reinterpret_cast<OutT*>(p.c) + m0 * p.ldc + n0, p.ldc, p.vec, smem);
}
template <class W, int CODE_A, bool B1D, typename OutT>
__global__ __launch_bounds__(W::THREADS, 2) void fp8_gemm_kernel(const Fp8GemmArgs p) {
  extern __shared__ __attribute__((aligned(16))) uint8_t smem[];
  int wg = blockIdx.x, quarter = 0;
  const int behind = (wg >> 3) - p.whole;
  if (behind >= 0) {
    wg = (wg & 7) + 8 * (p.whole + behind / 4);
    quarter = behind % 4;
  }
  int tm, tn;
  if (!fp8_tile_coords(wg, p.tiles_m, p.tiles_n, tm, tn)) return;
  int64_t m0 = (int64_t)tm * W::TM, n0 = (int64_t)tn * W::TN;
  if constexpr (W::TM == 256) {
    static_assert(W::THREADS == Split::THREADS && W::LDS >= Split::LDS, "");
    if (behind >= 0) {
      m0 += quarter / 2 * 128;
      n0 += quarter % 2 * 128;
      if (m0 < p.M && n0 < p.N) product<Split, CODE_A, B1D, OutT>(p, m0, n0, smem);
      return;
    }
  }
  product<W, CODE_A, B1D, OutT>(p, m0, n0, smem);
}

// An XCD's 32 compute units take 32 tiles of 256 x 256 at a time.  Where a last round would have 8 of them at most, these are cut into quarters, one round of workgroups
// whose halves take half of K each: 4 and 0.575 us for each 128 of K where a round of whole tiles takes 7.5 and 1.2 (4352 x 4096 x 4096: 95.3 -> 76.6 us; 4096 x 8704 x 4096:
// 155.5 -> 133.2).  Of 9 to 16 tiles, two such rounds, nothing is gained: 6400 x 6400 x 2048 89.5 -> 91.6.
int whole_tiles(int per_xcd) { return per_xcd > 32 && per_xcd % 32 <= 8 ? per_xcd / 32 * 32 : per_xcd; }

template <class W>
bool fits(int64_t M, int64_t N) { return product_below(FP8_MOST_TILES<W>, (M + W::TM - 1) / W::TM, (N + W::TN - 1) / W::TN); }

template <class W, int CODE_A, bool B1D, typename OutT>
int launch(Fp8GemmArgs& a, hipStream_t st) {
  ALTO_REQUIRE(fits<W>(a.M, a.N), "fp8_gemm: too many tiles for one launch");
  a.tiles_m = (int)((a.M + W::TM - 1) / W::TM);
  a.tiles_n = (int)((a.N + W::TN - 1) / W::TN);
  static LdsLimit limit;
  const int rc = limit.raise(reinterpret_cast<const void*>(&fp8_gemm_kernel<W, CODE_A, B1D, OutT>), W::LDS, "fp8_gemm");
  if (rc != ALTO_MXFP4_OK) return rc;
  const int per_xcd = (a.tiles_m * a.tiles_n + 7) / 8;
  a.whole = W::TM == 256 ? whole_tiles(per_xcd) : per_xcd;
  const int grid = 8 * (a.whole + 4 * (per_xcd - a.whole));
  hipLaunchKernelGGL((fp8_gemm_kernel<W, CODE_A, B1D, OutT>), dim3(grid), dim3(W::THREADS), W::LDS, st, a);
  return check_launch("fp8_gemm");
}
template <class W, int CODE_A>
int launch_types(Fp8GemmArgs& a, bool b1d, bool f32, hipStream_t st) {
  if (b1d) return f32 ? launch<W, CODE_A, true, float>(a, st) : launch<W, CODE_A, true, __bf16>(a, st);
  return f32 ? launch<W, CODE_A, false, float>(a, st) : launch<W, CODE_A, false, __bf16>(a, st);
}

template <int MT, int NT, int CODE_A, bool B1D, typename OutT>
__global__ __launch_bounds__(64 * FP8_ROWS_WAVES) void fp8_rows_kernel(const Fp8GemmArgs p) {
  __shared__ v4f_t sums[FP8_ROWS_WAVES * MT * NT * 64];
  const int64_t m0 = (int64_t)blockIdx.y * 16 * MT, n0 = (int64_t)blockIdx.x * 16 * NT;
  const Fp8RowsOperand A{p.a + m0 * p.lda, p.a_scales + (m0 >> p.a_shift) * p.a_ss_r, p.lda, p.a_ss_r, p.a_ss_k, (int)(p.M - m0 < 16 * MT ? p.M - m0 : 16 * MT), p.a_shift};
  const Fp8RowsOperand B{p.b + n0 * p.ldb, p.b_scales + (n0 >> p.b_shift) * p.b_ss_r, p.ldb, p.b_ss_r, p.b_ss_k, (int)(p.N - n0 < 16 * NT ? p.N - n0 : 16 * NT), p.b_shift};
  fp8_rows_product<MT, NT, CODE_A, B1D>(A, B, (int)p.K, reinterpret_cast<OutT*>(p.c) + m0 * p.ldc + n0, p.ldc, sums);
}
template <int MT, int NT, int CODE_A, bool B1D, typename OutT>
int launch_rows(const Fp8GemmArgs& a, hipStream_t st) {
  const int64_t gx = (a.N + 16 * NT - 1) / (16 * NT), gy = (a.M + 16 * MT - 1) / (16 * MT);
  ALTO_REQUIRE(product_below(1ll << 23, gx, gy), "fp8_gemm: too many tiles for one launch");   // (its threads are counted in 32 bits)
  hipLaunchKernelGGL((fp8_rows_kernel<MT, NT, CODE_A, B1D, OutT>), dim3((unsigned)gx, (unsigned)gy), dim3(64 * FP8_ROWS_WAVES), 0, st, a);
  return check_launch("fp8_gemm");
}
template <int MT, int NT, int CODE_A>
int launch_rows_types(const Fp8GemmArgs& a, bool b1d, bool f32, hipStream_t st) {
  if (b1d) return f32 ? launch_rows<MT, NT, CODE_A, true, float>(a, st) : launch_rows<MT, NT, CODE_A, true, __bf16>(a, st);
  return f32 ? launch_rows<MT, NT, CODE_A, false, float>(a, st) : launch_rows<MT, NT, CODE_A, false, __bf16>(a, st);
}
template <int CODE_A>
int launch_few_rows(const Fp8GemmArgs& a, int mt, int nt, bool b1d, bool f32, hipStream_t st) {
  if (mt == 1) return nt == 1 ? launch_rows_types<1, 1, CODE_A>(a, b1d, f32, st) : launch_rows_types<1, 2, CODE_A>(a, b1d, f32, st);
  if (mt == 2) return nt == 1 ? launch_rows_types<2, 1, CODE_A>(a, b1d, f32, st) : launch_rows_types<2, 2, CODE_A>(a, b1d, f32, st);
  return launch_rows_types<4, 2, CODE_A>(a, b1d, f32, st);
}

}  // namespace

static int fp8_gemm(const alto_mxfp4_fp8_gemm_t& p, hipStream_t st) {
  ALTO_REQUIRE(p.a_code == ALTO_FP8_E4M3 || p.a_code == ALTO_FP8_E5M2, "fp8_gemm: code %d is neither E4M3 (0) nor E5M2 (1)", p.a_code);
  ALTO_REQUIRE(p.c_dtype == ALTO_DT_BF16 || p.c_dtype == ALTO_DT_F32, "fp8_gemm: dtype %d is neither bf16 (0) nor f32 (1)", p.c_dtype);
  ALTO_REQUIRE(p.M >= 0 && p.N >= 0 && p.K >= 0 && p.M < (1ll << 31) && p.N < (1ll << 31) && p.K <= (1ll << 22) - 16, "fp8_gemm: size out of range");
  if (p.M == 0 || p.N == 0) return ALTO_MXFP4_OK;
  const int64_t size = p.c_dtype == ALTO_DT_BF16 ? 2 : 4, k16 = (p.K + 15) / 16 * 16;
  ALTO_REQUIRE(p.c && (p.K == 0 || (p.a && p.b && p.a_scales && p.b_scales)), "fp8_gemm: null pointer");
  ALTO_REQUIRE(((uintptr_t)p.a | (uintptr_t)p.b) % 16 == 0 && ((uintptr_t)p.a_scales | (uintptr_t)p.b_scales) % 4 == 0 && (uintptr_t)p.c % (uintptr_t)size == 0, "fp8_gemm: misaligned pointer");
  ALTO_REQUIRE(p.lda >= 0 && p.lda % 16 == 0 && p.lda < (1ll << 22) && (p.M == 1 || p.lda >= k16) && p.ldb >= 0 && p.ldb % 16 == 0 && p.ldb < (1ll << 22) && (p.N == 1 || p.ldb >= k16),
               "fp8_gemm: rows of codes must be multiples of 16 bytes, at least K and below 2^22 apart");
  for (const int64_t s : {p.a_ss_r, p.b_ss_r}) ALTO_REQUIRE(s >= 0 && s < (1ll << 21), "fp8_gemm: scales of neighbouring rows are too far apart");
  for (const int64_t s : {p.a_ss_k, p.b_ss_k}) ALTO_REQUIRE(s >= 0 && s < (1ll << 40), "fp8_gemm: strides of scales must be non-negative");
  ALTO_REQUIRE(p.ldc >= 0 && p.ldc < (1ll << 40) && (p.M == 1 || p.ldc >= p.N), "fp8_gemm: rows of the result overlap");
  Fp8GemmArgs a{(const uint8_t*)p.a, (const uint8_t*)p.b, p.a_scales, p.b_scales, p.c, p.M, p.N, p.K, p.lda, p.ldb, p.a_ss_r, p.a_ss_k, p.b_ss_r, p.b_ss_k, p.ldc,
                p.a_is_2d ? 7 : 0, p.b_is_2d ? 7 : 0, 0, 0, 0, (uintptr_t)p.c % 16 == 0 && p.ldc * size % 16 == 0};
  const bool f32 = p.c_dtype == ALTO_DT_F32, b1d = !p.b_is_2d;
  const int64_t large = ((p.M + 255) / 256) * ((p.N + 255) / 256), small = ((p.M + 127) / 128) * ((p.N + 127) / 128);
  // 256 x 256 or 128 x 128, by what either was measured to take (us).  A round of at most 256 of the first: 7.5 and 1.2 to 1.45 for each 128 of K, and the quarters of a last
  // one.  The second, 512 at a time: 7 and 0.95 for each 128 of K, then 3, and 2.5 and 1.11 for each 128 of K and round, the last one no less than 0.55 of one.  Within 12 %
  // over these (first, second): 1500 x 4096 x 4096 46.5, 33.0; 2304 x 4096 x 2048 27.7, 33.5; 3000 x 4096 x 2048 29.4, 34.6; 2048 x 4096 x 4096 46.1, 36.5; 5000 x 5000 x
  // 1024 40.0, 45.0; 8192 x 8192 x 256 42.5, 40.9; 2048 x 14336 x 4096 113, 137.  (All with scales of B for 128 x 128.  With one for each of its rows stages take longer on either side, 1.75
  // to 1.97 of the first: the same rule serves, its pairs are not measured.)
  const double kb = (double)((p.K + 127) / 128), share = large < 256 ? (double)large / 256 : 1.0;
  const int per_xcd = (int)((large + 7) / 8 < 1 << 20 ? (large + 7) / 8 : 1 << 20), whole = whole_tiles(per_xcd);
  const double of_large = (double)((whole + 31) / 32) * (7.5 + kb * (1.2 + 0.25 * share)) + (per_xcd == whole ? 0.0 : 4.0 + 0.575 * kb);
  const double rest = (double)(small % 512) / 512, rounds = (double)(small / 512) + (rest > 0.0 && rest < 0.55 ? 0.55 : rest);
  const double of_small = small <= 512 ? 7.0 + kb * (small > 458 ? 0.95 * (double)small / 512 : 0.85) : 3.0 + rounds * (2.5 + 1.11 * kb);
  // (more of the second than one launch takes are no choice)
  if (of_large <= of_small || !fits<Small>(p.M, p.N)) return p.a_code == ALTO_FP8_E4M3 ? launch_types<Large, ALTO_FP8_E4M3>(a, b1d, f32, st) : launch_types<Large, ALTO_FP8_E5M2>(a, b1d, f32, st);
  if (small <= 256) {
    // Few tiles (of more, as a row by more than 32768 columns makes, none of these was measured): 128 x 128 with K in halves, 64 x 64 with K in quarters, or the kernel for few rows, by what each was measured to take (us; within 20 % over 1 to 768 rows, N
    // and K from 512 to 14336).  The first: 4, and 0.9 to 1.15 for each 256 of K.  The second: 3.2 and 1.06 for each 512 of K and 256 tiles, and no less than 3 and the operands at
    // 4.2 TB/s.  The third: 2.5 and, 256 workgroups at a time, their reads at 31 GB/s x 1000 each, no less than the operands at 6.3 TB/s.  (First, second, third: 32 x 4096 x 4096 17.1,
    // 10.7, 8.2; 32 x 14336 x 4096 22.4, 17.3, 19.9; 64 x 14336 x 4096 22.8, 17.9, 22.6; 128 x 4096 x 4096 17.7, 11.2, 14.7; 256 x 4096 x 4096 22.0, 11.5, -; 128 x 14336 x 4096 23.3, 28.5, -; 256 x 1024 x 14336
    // 63, 34, 27.9; 512 x 4096 x 4096 22.4, 24.2, -.)
    const double operands = (double)(p.M + p.N) * (double)p.K;
    const double split = 4.0 + (double)((p.K + 255) / 256) * (0.9 + 0.25 * (double)small / 256);
    const double tiles_64 = (double)((p.M + 63) / 64) * (double)((p.N + 63) / 64), rounds_64 = (double)(((int64_t)tiles_64 + 255) / 256);
    double four = rounds_64 * (3.2 + 1.06 * (double)((p.K + 511) / 512));
    if (four < 3.0 + operands / 4.2e6) four = 3.0 + operands / 4.2e6;
    double best = four < split ? four : split;
    int mt = 0, nt = 0;
    for (const auto& [m, n] : {std::pair{1, 1}, {1, 2}, {2, 1}, {2, 2}, {4, 2}}) {
      const int64_t groups = ((p.M + 16 * m - 1) / (16 * m)) * ((p.N + 16 * n - 1) / (16 * n));   // (M and N are at most 32768 here)
      const double each = (double)((p.M < 16 * m ? p.M : 16 * m) + 16 * n) * (double)p.K;
      double us = (double)((groups + 255) / 256) * each / 31e3;
      if (us < operands / 6.3e6) us = operands / 6.3e6;
      if (2.5 + us < best) {
        best = 2.5 + us;
        mt = m;
        nt = n;
      }
    }
    if (mt != 0) return p.a_code == ALTO_FP8_E4M3 ? launch_few_rows<ALTO_FP8_E4M3>(a, mt, nt, b1d, f32, st) : launch_few_rows<ALTO_FP8_E5M2>(a, mt, nt, b1d, f32, st);
    if (four < split) return p.a_code == ALTO_FP8_E4M3 ? launch_types<Four, ALTO_FP8_E4M3>(a, b1d, f32, st) : launch_types<Four, ALTO_FP8_E5M2>(a, b1d, f32, st);
    return p.a_code == ALTO_FP8_E4M3 ? launch_types<Split, ALTO_FP8_E4M3>(a, b1d, f32, st) : launch_types<Split, ALTO_FP8_E5M2>(a, b1d, f32, st);
  }
  return p.a_code == ALTO_FP8_E4M3 ? launch_types<Small, ALTO_FP8_E4M3>(a, b1d, f32, st) : launch_types<Small, ALTO_FP8_E5M2>(a, b1d, f32, st);
}

}  // namespace alto

extern "C" int alto_mxfp4_fp8_gemm(const alto_mxfp4_fp8_gemm_t* p, void* stream) {
  ALTO_REQUIRE(p, "fp8_gemm: null pointer");
  return alto::fp8_gemm(*p, (hipStream_t)stream);
}
