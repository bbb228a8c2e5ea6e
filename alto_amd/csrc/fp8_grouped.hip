// Products of 8-bit floating-point operands with a scale for each block of 128 (fp8_tile.h): rows grouped by expert, and their weight gradients.
//
// No list of tiles is built ahead: the number of a tile's rows among all groups' tiles is the workgroup's, and every wave finds the rows behind it with one
// scan over the boundaries (64 groups at a time, fp8.h), which the tile's first loads would wait for longer.
//
// Measured, 32 experts of 5760 x 2880, groups from 1/4 to 1/130 of all rows: 65536 rows 1160 us (1870 TFLOP/s), their input gradients 1100 (1980), their weight gradients 1320
// to 1365 (1600 to 1650; a scale for each row of both operands, where the tile alone reaches 2026); 96 rows, 85 of them routed, 106 us, 4.6 TB/s of the weights that
// they meet.  By expert a tile's fixed 7.5 us weigh more than in one long product: K is 23 blocks of 128, and of the weight gradients 16 on average.
#include "fp8_rows.h"
#include "fp8_tile.h"

namespace alto {
namespace {

typedef Fp8Tile<2, 4, 8> Large;
typedef Fp8Tile<2, 2, 4> Small;

struct Fp8GroupedArgs {
  const uint8_t *a, *w;
  const float *a_scales, *w_scales;
  void* c;
  const int32_t* offs;
  int64_t M, N, K, lda, a_ss_r, a_ss_k, w_se, ldw, ws_e, ws_r, ws_k, ldc;
  int groups, w_shift, tiles_n, vec;
};

int64_t used_pieces(const Fp8GroupedArgs& a, int piece) {   // at most so many hold a row
  const int64_t n = most_pieces(a.M, a.groups, piece);
  return n < a.M ? n : a.M;
}

template <class W, int CODE_A, bool B1D, typename OutT>
__global__ __launch_bounds__(W::THREADS, 2) void fp8_grouped_kernel(const Fp8GroupedArgs p) {
  extern __shared__ __attribute__((aligned(16))) uint8_t smem[];
  int tn;
  Segment seg;
  if (!find_tile(p.offs, p.groups, p.M, W::TM, blockIdx.x, p.tiles_n, fp8_tile_coords, seg, tn)) return;
  const int rows = (int)(seg.hi - seg.lo);
  const int64_t n0 = (int64_t)tn * W::TN;
  const int cols = (int)(p.N - n0 < W::TN ? p.N - n0 : W::TN);
  Fp8TileArgs t;
  const int64_t e = seg.group < 0 ? 0 : seg.group;
  t.A = {p.a + seg.lo * p.lda, p.a_scales + seg.lo * p.a_ss_r, p.lda, p.a_ss_r, p.a_ss_k, rows, 0};
  t.B = {p.w + e * p.w_se + n0 * p.ldw, p.w_scales + e * p.ws_e + (n0 >> p.w_shift) * p.ws_r, p.ldw, p.ws_r, p.ws_k, cols, p.w_shift};
  t.K = seg.group < 0 ? 0 : p.K;   // rows of no group: zeros
  fp8_tile_product<W, CODE_A, B1D>(t, reinterpret_cast<OutT*>(p.c) + seg.lo * p.ldc + n0, p.ldc, p.vec, smem);
}

template <class W>
bool fits(const Fp8GroupedArgs& a) { return product_below(FP8_MOST_TILES<W>, used_pieces(a, W::TM), (a.N + W::TN - 1) / W::TN); }

template <class W, int CODE_A, bool B1D, typename OutT>
int launch(Fp8GroupedArgs& a, hipStream_t st) {
  ALTO_REQUIRE(fits<W>(a), "fp8_grouped_gemm: too many tiles for one launch");
  const int64_t tiles_m = used_pieces(a, W::TM);
  a.tiles_n = (int)((a.N + W::TN - 1) / W::TN);
  static LdsLimit limit;
  const int rc = limit.raise(reinterpret_cast<const void*>(&fp8_grouped_kernel<W, CODE_A, B1D, OutT>), W::LDS, "fp8_grouped_gemm");
  if (rc != ALTO_MXFP4_OK) return rc;
  const int grid = ((int)tiles_m * a.tiles_n + 7) / 8 * 8;
  hipLaunchKernelGGL((fp8_grouped_kernel<W, CODE_A, B1D, OutT>), dim3(grid), dim3(W::THREADS), W::LDS, st, a);
  return check_launch("fp8_grouped_gemm");
}
template <class W, int CODE_A>
int launch_types(Fp8GroupedArgs& a, bool b1d, bool f32, hipStream_t st) {
  if (b1d) return f32 ? launch<W, CODE_A, true, float>(a, st) : launch<W, CODE_A, true, __bf16>(a, st);
  return f32 ? launch<W, CODE_A, false, float>(a, st) : launch<W, CODE_A, false, __bf16>(a, st);
}

template <int MT, int NT, int CODE_A, bool B1D, typename OutT>
__global__ __launch_bounds__(64 * FP8_ROWS_WAVES) void fp8_grouped_rows_kernel(const Fp8GroupedArgs p) {
  __shared__ v4f_t sums[FP8_ROWS_WAVES * MT * NT * 64];
  const Segment seg = find_piece(p.offs, p.groups, p.M, 16 * MT, blockIdx.x / p.tiles_n);
  const int rows = (int)(seg.hi - seg.lo);
  if (rows <= 0) return;
  const int64_t n0 = (int64_t)(blockIdx.x % p.tiles_n) * 16 * NT, e = seg.group < 0 ? 0 : seg.group;
  const Fp8RowsOperand A{p.a + seg.lo * p.lda, p.a_scales + seg.lo * p.a_ss_r, p.lda, p.a_ss_r, p.a_ss_k, rows, 0};
  const Fp8RowsOperand B{p.w + e * p.w_se + n0 * p.ldw, p.w_scales + e * p.ws_e + (n0 >> p.w_shift) * p.ws_r, p.ldw, p.ws_r, p.ws_k, (int)(p.N - n0 < 16 * NT ? p.N - n0 : 16 * NT), p.w_shift};
  fp8_rows_product<MT, NT, CODE_A, B1D>(A, B, seg.group < 0 ? 0 : (int)p.K, reinterpret_cast<OutT*>(p.c) + seg.lo * p.ldc + n0, p.ldc, sums);   // (rows of no group: zeros)
}
template <int MT, int NT, int CODE_A, bool B1D, typename OutT>
int launch_rows(Fp8GroupedArgs& a, hipStream_t st) {
  const int64_t tiles_m = used_pieces(a, 16 * MT);
  a.tiles_n = (int)((a.N + 16 * NT - 1) / (16 * NT));
  ALTO_REQUIRE(product_below(1ll << 23, tiles_m, a.tiles_n), "fp8_grouped_gemm: too many tiles for one launch");   // (its threads are counted in 32 bits)
  hipLaunchKernelGGL((fp8_grouped_rows_kernel<MT, NT, CODE_A, B1D, OutT>), dim3((unsigned)(tiles_m * a.tiles_n)), dim3(64 * FP8_ROWS_WAVES), 0, st, a);
  return check_launch("fp8_grouped_gemm");
}
template <int MT, int NT, int CODE_A>
int launch_rows_types(Fp8GroupedArgs& a, bool b1d, bool f32, hipStream_t st) {
  if (b1d) return f32 ? launch_rows<MT, NT, CODE_A, true, float>(a, st) : launch_rows<MT, NT, CODE_A, true, __bf16>(a, st);
  return f32 ? launch_rows<MT, NT, CODE_A, false, float>(a, st) : launch_rows<MT, NT, CODE_A, false, __bf16>(a, st);
}

struct Fp8WeightsArgs {
  const uint8_t *go, *x;
  const float *go_scales, *x_scales;
  void* dw;
  const int32_t* offs;
  int64_t tokens, N, K, go_ld, x_ld, go_ss, x_ss, dw_se, ld_dw;
  int groups, tiles_n, tiles_k, vec;
};

template <class W, int CODE_A, typename OutT>
__global__ __launch_bounds__(W::THREADS, 2) void fp8_grouped_weights_kernel(const Fp8WeightsArgs p) {
  extern __shared__ __attribute__((aligned(16))) uint8_t smem[];
  int tn, tk;
  const int e = blockIdx.y;
  if (!fp8_tile_coords(blockIdx.x, p.tiles_n, p.tiles_k, tn, tk)) return;
  const GroupSpan span = find_group(p.offs, p.groups, 0x7FFFFFFF, 128, e);
  int64_t blocks = (span.hi - span.lo + 127) / 128;   // (zeros behind the group's last token)
  blocks = span.piece0 + blocks <= p.tokens / 128 ? blocks : span.piece0 < p.tokens / 128 ? p.tokens / 128 - span.piece0 : 0;
  const int64_t n0 = (int64_t)tn * W::TM, k0 = (int64_t)tk * W::TN, t0 = blocks > 0 ? span.piece0 * 128 : 0;
  Fp8TileArgs t;
  t.A = {p.go + n0 * p.go_ld + t0, p.go_scales + n0 + t0 / 128 * p.go_ss, p.go_ld, 1, p.go_ss, (int)(p.N - n0 < W::TM ? p.N - n0 : W::TM), 0};
  t.B = {p.x + k0 * p.x_ld + t0, p.x_scales + k0 + t0 / 128 * p.x_ss, p.x_ld, 1, p.x_ss, (int)(p.K - k0 < W::TN ? p.K - k0 : W::TN), 0};
  t.K = blocks * 128;
  fp8_tile_product<W, CODE_A, true>(t, reinterpret_cast<OutT*>(p.dw) + e * p.dw_se + n0 * p.ld_dw + k0, p.ld_dw, p.vec, smem);
}

template <class W, int CODE_A, typename OutT>
int launch_weights(Fp8WeightsArgs& a, hipStream_t st) {
  a.tiles_n = (int)((a.N + W::TM - 1) / W::TM);
  a.tiles_k = (int)((a.K + W::TN - 1) / W::TN);
  ALTO_REQUIRE(product_below(FP8_MOST_TILES<W>, a.tiles_n, a.tiles_k), "fp8_grouped_gemm_weights: too many tiles for one launch");
  static LdsLimit limit;
  const int rc = limit.raise(reinterpret_cast<const void*>(&fp8_grouped_weights_kernel<W, CODE_A, OutT>), W::LDS, "fp8_grouped_gemm_weights");
  if (rc != ALTO_MXFP4_OK) return rc;
  const dim3 grid((a.tiles_n * a.tiles_k + 7) / 8 * 8, a.groups);
  hipLaunchKernelGGL((fp8_grouped_weights_kernel<W, CODE_A, OutT>), grid, dim3(W::THREADS), W::LDS, st, a);
  return check_launch("fp8_grouped_gemm_weights");
}
template <class W>
int launch_weights_types(Fp8WeightsArgs& a, int code, bool f32, hipStream_t st) {
  if (code == ALTO_FP8_E4M3) return f32 ? launch_weights<W, ALTO_FP8_E4M3, float>(a, st) : launch_weights<W, ALTO_FP8_E4M3, __bf16>(a, st);
  return f32 ? launch_weights<W, ALTO_FP8_E5M2, float>(a, st) : launch_weights<W, ALTO_FP8_E5M2, __bf16>(a, st);
}

}  // namespace

static int fp8_grouped_gemm(const alto_mxfp4_fp8_grouped_gemm_t& p, hipStream_t st) {
  ALTO_REQUIRE(p.a_code == ALTO_FP8_E4M3 || p.a_code == ALTO_FP8_E5M2, "fp8_grouped_gemm: code %d is neither E4M3 (0) nor E5M2 (1)", p.a_code);
  ALTO_REQUIRE(p.c_dtype == ALTO_DT_BF16 || p.c_dtype == ALTO_DT_F32, "fp8_grouped_gemm: dtype %d is neither bf16 (0) nor f32 (1)", p.c_dtype);
  ALTO_REQUIRE(p.M >= 0 && p.N >= 0 && p.K >= 0 && p.M < (1ll << 31) && p.N < (1ll << 31) && p.K <= (1ll << 22) - 16, "fp8_grouped_gemm: size out of range");
  ALTO_REQUIRE(p.groups >= 1 && p.groups < 65536, "fp8_grouped_gemm: %d groups, 1 to 65535 are taken", p.groups);
  if (p.M == 0 || p.N == 0) return ALTO_MXFP4_OK;
  const int64_t size = p.c_dtype == ALTO_DT_BF16 ? 2 : 4, k16 = (p.K + 15) / 16 * 16;
  ALTO_REQUIRE(p.c && p.offs && (p.K == 0 || (p.a && p.w && p.a_scales && p.w_scales)), "fp8_grouped_gemm: null pointer");
  ALTO_REQUIRE(((uintptr_t)p.a | (uintptr_t)p.w) % 16 == 0 && ((uintptr_t)p.a_scales | (uintptr_t)p.w_scales | (uintptr_t)p.offs) % 4 == 0 && (uintptr_t)p.c % (uintptr_t)size == 0,
               "fp8_grouped_gemm: misaligned pointer");
  ALTO_REQUIRE(p.lda >= 0 && p.lda % 16 == 0 && p.lda < (1ll << 22) && (p.M == 1 || p.lda >= k16) && p.ldw >= 0 && p.ldw % 16 == 0 && p.ldw < (1ll << 22) && (p.N == 1 || p.ldw >= k16),
               "fp8_grouped_gemm: rows of codes must be multiples of 16 bytes, at least K and below 2^22 apart");
  ALTO_REQUIRE(p.w_se >= 0 && p.w_se % 16 == 0 && p.w_se < (1ll << 45), "fp8_grouped_gemm: the experts' codes must be multiples of 16 bytes apart");
  for (const int64_t s : {p.a_ss_r, p.ws_r}) ALTO_REQUIRE(s >= 0 && s < (1ll << 21), "fp8_grouped_gemm: scales of neighbouring rows are too far apart");
  for (const int64_t s : {p.a_ss_k, p.ws_k, p.ws_e}) ALTO_REQUIRE(s >= 0 && s < (1ll << 40), "fp8_grouped_gemm: strides of scales must be non-negative");
  ALTO_REQUIRE(p.ldc >= 0 && p.ldc < (1ll << 40) && (p.M == 1 || p.ldc >= p.N), "fp8_grouped_gemm: rows of the result overlap");
  Fp8GroupedArgs a{(const uint8_t*)p.a, (const uint8_t*)p.w, p.a_scales, p.w_scales, p.c, p.offs, p.M, p.N, p.K, p.lda, p.a_ss_r, p.a_ss_k, p.w_se, p.ldw, p.ws_e, p.ws_r, p.ws_k, p.ldc,
                   p.groups, p.w_is_2d ? 7 : 0, 0, (uintptr_t)p.c % 16 == 0 && p.ldc * size % 16 == 0};
  const bool f32 = p.c_dtype == ALTO_DT_F32, b1d = !p.w_is_2d;
  // Few rows a group: 16 rows at a time, K split over the waves, the longer K is the more rows (16 rows, 128 x 128, us: 32 experts of 5760 x 2880, 64 rows 98.8, 102.4, 96 rows
  // 111, 106; of 2880 x 5760, 128 rows 108.6, 120.4, 256 rows 125, 120.5; 64 of 512 x 2048, 64 rows 11.5, 18.2; 8 of 4096 x 1024, 8 rows 9.9, 9.1).
  if (p.M * 1024 < (int64_t)p.groups * (p.K < 8192 ? p.K : 8192) && product_below(1ll << 23, used_pieces(a, 16), (p.N + 31) / 32)) return p.a_code == ALTO_FP8_E4M3 ? launch_rows_types<1, 2, ALTO_FP8_E4M3>(a, b1d, f32, st) : launch_rows_types<1, 2, ALTO_FP8_E5M2>(a, b1d, f32, st);
  // (256 x 256, 128 x 128, us: 32 experts of 5760 x 2880, 4096 rows 183, 163, 8192 rows 232, 232, 16384 rows 341, 396; 8 of 4096 x 1024, 1024 rows 18.0, 13.5, 2048 rows 18.7, 22.0; fewer than 8
  // groups are not measured, and tiles whose waves share K, which one weight's products of few tiles have, are not built by group;
  // more of either than one launch takes are no choice)
  const bool large = p.M >= 256ll * p.groups && p.N > 128 ? fits<Large>(a) || !fits<Small>(a) : !fits<Small>(a);
  if (large) return p.a_code == ALTO_FP8_E4M3 ? launch_types<Large, ALTO_FP8_E4M3>(a, b1d, f32, st) : launch_types<Large, ALTO_FP8_E5M2>(a, b1d, f32, st);
  return p.a_code == ALTO_FP8_E4M3 ? launch_types<Small, ALTO_FP8_E4M3>(a, b1d, f32, st) : launch_types<Small, ALTO_FP8_E5M2>(a, b1d, f32, st);
}

static int fp8_grouped_gemm_weights(const alto_mxfp4_fp8_grouped_gemm_weights_t& p, hipStream_t st) {
  ALTO_REQUIRE(p.go_code == ALTO_FP8_E4M3 || p.go_code == ALTO_FP8_E5M2, "fp8_grouped_gemm_weights: code %d is neither E4M3 (0) nor E5M2 (1)", p.go_code);
  ALTO_REQUIRE(p.dw_dtype == ALTO_DT_BF16 || p.dw_dtype == ALTO_DT_F32, "fp8_grouped_gemm_weights: dtype %d is neither bf16 (0) nor f32 (1)", p.dw_dtype);
  ALTO_REQUIRE(p.groups >= 1 && p.groups < 65536, "fp8_grouped_gemm_weights: %d groups, 1 to 65535 are taken", p.groups);
  ALTO_REQUIRE(p.tokens >= 0 && p.tokens % 128 == 0 && p.tokens < (1ll << 22) && p.N >= 0 && p.K >= 0 && p.N < (1ll << 31) && p.K < (1ll << 31), "fp8_grouped_gemm_weights: size out of range");
  if (p.N == 0 || p.K == 0) return ALTO_MXFP4_OK;
  const int64_t tokens = p.tokens, size = p.dw_dtype == ALTO_DT_BF16 ? 2 : 4;
  ALTO_REQUIRE(p.dw && p.offs && (tokens == 0 || (p.go && p.x && p.go_scales && p.x_scales)), "fp8_grouped_gemm_weights: null pointer");
  ALTO_REQUIRE(((uintptr_t)p.go | (uintptr_t)p.x) % 16 == 0 && ((uintptr_t)p.go_scales | (uintptr_t)p.x_scales | (uintptr_t)p.offs) % 4 == 0 && (uintptr_t)p.dw % (uintptr_t)size == 0,
               "fp8_grouped_gemm_weights: misaligned pointer");
  ALTO_REQUIRE(p.go_ld >= 0 && p.go_ld % 16 == 0 && p.go_ld < (1ll << 22) && (p.N == 1 || p.go_ld >= tokens) && p.x_ld >= 0 && p.x_ld % 16 == 0 && p.x_ld < (1ll << 22) && (p.K == 1 || p.x_ld >= tokens),
               "fp8_grouped_gemm_weights: rows of codes must be multiples of 16 bytes, at least all tokens and below 2^22 apart");
  for (const int64_t s : {p.go_ss, p.x_ss, p.dw_se, p.ld_dw}) ALTO_REQUIRE(s >= 0 && s < (1ll << 40), "fp8_grouped_gemm_weights: strides must be non-negative");
  ALTO_REQUIRE((p.N == 1 || p.ld_dw >= p.K) && (p.groups == 1 || p.dw_se >= (p.N - 1) * p.ld_dw + p.K), "fp8_grouped_gemm_weights: rows of the result overlap");
  Fp8WeightsArgs a{(const uint8_t*)p.go, (const uint8_t*)p.x, p.go_scales, p.x_scales, p.dw, p.offs, p.tokens, p.N, p.K, p.go_ld, p.x_ld, p.go_ss, p.x_ss, p.dw_se, p.ld_dw,
                   p.groups, 0, 0, (uintptr_t)p.dw % 16 == 0 && p.ld_dw * size % 16 == 0 && p.dw_se * size % 16 == 0};
  const bool f32 = p.dw_dtype == ALTO_DT_F32;
  // 256 x 256 where a group has enough such tiles to spread over the chip, however long it is; a group of few tiles may be the longest by far, and more of them shorten
  // it (256 x 256, 128 x 128, us; 2048 tokens a group, the longest 8 times as many or more: 8 of 4096 x 4096 302, 354; 32 of 5760 x 2880 1366, 1497; 8 of 4096 x 1024 104.5,
  // 97.8; 64 of 512 x 2048 400, 293; 512 tokens: 121, 132; 495, 529; 37.4, 37.2; 102, 85).
  const int64_t each = ((p.N + 255) / 256) * ((p.K + 255) / 256);
  if (each >= 128 && each * p.groups >= 200) return launch_weights_types<Large>(a, p.go_code, f32, st);
  return launch_weights_types<Small>(a, p.go_code, f32, st);
}

}  // namespace alto

extern "C" int alto_mxfp4_fp8_grouped_gemm(const alto_mxfp4_fp8_grouped_gemm_t* p, void* stream) {
  ALTO_REQUIRE(p, "fp8_grouped_gemm: null pointer");
  return alto::fp8_grouped_gemm(*p, (hipStream_t)stream);
}
extern "C" int alto_mxfp4_fp8_grouped_gemm_weights(const alto_mxfp4_fp8_grouped_gemm_weights_t* p, void* stream) {
  ALTO_REQUIRE(p, "fp8_grouped_gemm_weights: null pointer");
  return alto::fp8_grouped_gemm_weights(*p, (hipStream_t)stream);
}
