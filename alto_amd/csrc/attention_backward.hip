// Gradients of the MXFP4 attention with respect to Q, K and V (gfx950).
//
// With S_ij = sm_scale Q_i . K_j + bias_ij - slope |i + Sk - Sq - j| on the values that the codes stand for, and the forward's log-sum-exp:
//   P_ij = exp(S_ij - lse_i)   (0 where the mask hides j, and in a row that sees no key),   D_i = dO_i . O_i,
//   dV_j = sum_i P_ij dO_i,   dS_ij = P_ij (dO_i . V_j - D_i),   dQ_i = sm_scale sum_j dS_ij K_j,   dK_j = sm_scale sum_i dS_ij Q_i.
// The roundings of Q, K, V and P to FP4 are passed straight through; lse and O are the forward's, which sums quantized probabilities: P sums to one
// and D is the mean of dO . V only up to their rounding.  The scores are recomputed on the FP4 pipe from the forward's codes;
// the other products have a factor that is not on the FP4 grid (P, dS, dO) and run in bf16, in which the codes' values are exact.  P and
// dS are rounded to bf16 as factors: half a step, 2^-8 of a value at most, so that a sum is off by at most 2^-8 of the sum of its terms' magnitudes
// (of the sum itself, which may cancel, by more; all gradients together by 2.4e-3 of their size, their own rounding alone 1.7e-3).  Scores,
// probabilities, dS before that, D and all sums are fp32.
//
// Two launches, or three.  This file's preparation reads every operand once and writes what the main kernel's many workgroups read over and
// over in the order in which they read it: D and lse, the scale bytes, and tiles of K's and V's values and of dO in bf16.  (A copy of dO costs 2
// bytes read and written an element once; read with the caller's strides it would be 64-byte pieces, for every key block anew.)  The main
// kernel has dK and dV by blocks of keys and dQ by blocks of rows: the one needs a sum over rows, the other over keys, so each recomputes P
// and every gradient is summed by one wave in a fixed order, with no atomics: the results do not change from run to run.  Where the lists of
// a few key blocks would outlast the rest they are cut, and a third kernel adds the parts, in fp32 and in their order.
//
// The preparation is bound by HBM (6 bytes an element of dO, 2.5 one of K and V): 79 us for 4 x 2048 tokens, 64 / 8 heads of 128, 5.6 TB/s.
#include <algorithm>
#include <memory>
#include <new>

#include "attention_backward.h"

namespace alto {
namespace {

struct PrepareArgs {
  const uint8_t *qs, *k, *ks, *vt, *vs;
  const __bf16 *dout, *out;
  const float *lse, *alibi;
  float sm_scale;
  int64_t alibi_sb, alibi_sh, do_sb, do_sh, do_ss, o_sb, o_sh, o_ss, l_sb, l_sh, l_ss;
  int Hq, Hk, Sq, Sk, D, Dv;
  int q_tiles;   // B Hq Sq / 32
  QRecord* q_records;
  KRecord* k_records;
  v4i_t *k_rows, *v_rows, *g_rows;
};

// The scale bytes of a tile of Q or K in the order of the score products
__device__ __forceinline__ void order_scales(const uint8_t* scales, int64_t tile, int bands, uint8_t* ordered) {
  const int tid = threadIdx.x, c = 2 * (tid & 3) + (tid >> 2);
  if (tid < 8) ordered[tid] = c < bands ? scales[tile * bands + c] : 127;
}

// The values of a tile of K
__device__ __forceinline__ void decode_tile(const uint8_t* codes, const uint8_t* scales, int64_t tile, int D, v4i_t* rows) {
  const int tid = threadIdx.x;
  const uint8_t* s = scales + tile * (D / 32);
  const uint32_t* from = reinterpret_cast<const uint32_t*>(codes + tile * 16 * D);
  v4i_t* to = rows + tile * 4 * D;
  for (int i = tid; i < 4 * D; i += 256) {
    const int p = i >> 5, row = (i & 31) ^ ((p & 3) << 2);   // piece i of the tile
    to[i] = decode8(from[row * (D / 8) + p], e8m0_value(s[p >> 2]));
  }
}

// One workgroup: 32 query rows (dO, their statistics, the scales of Q), or 32 keys of K and V.
__global__ __launch_bounds__(256) void attn_bwd_prepare_kernel(const PrepareArgs a) {
  __shared__ __align__(16) uint32_t turned[4][32 * 20];   // one 32 x 32 block of V a wave, rows of 64 bytes 80 apart; or a tile of dO
  const int tid = threadIdx.x;
  int64_t tile = blockIdx.x;
  if (tile < a.q_tiles) {
    order_scales(a.qs, tile, a.D / 32, a.q_records[tile].scales);
    v4i_t* const grad = reinterpret_cast<v4i_t*>(turned);
    const int r = tid >> 3, c = tid & 7;
    const int64_t row = tile * 32 + r, bh = row / a.Sq;
    const int64_t b = bh / a.Hq, h = bh % a.Hq, i = row % a.Sq;
    if (tid == 0) a.q_records[tile].slope = a.alibi ? -a.alibi[b * a.alibi_sb + h * a.alibi_sh] / a.sm_scale : 0.0f;
    const v4i_t* go = reinterpret_cast<const v4i_t*>(a.dout + b * a.do_sb + h * a.do_sh + i * a.do_ss);
    const v4i_t* o = reinterpret_cast<const v4i_t*>(a.out + b * a.o_sb + h * a.o_sh + i * a.o_ss);
    const float l = a.lse[b * a.l_sb + h * a.l_sh + i * a.l_ss];
    const bool none = l == -__builtin_inff();   // a row that sees no key: it gives nothing, whatever the forward left in O and whatever dO holds
    float d = 0.0f;
    for (int p = c; p < a.Dv / 8; p += 8) {
      const v4i_t x = none ? v4i_t{0, 0, 0, 0} : go[p], y = o[p];
      grad[tile_piece(r, p)] = x;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        d = __builtin_fmaf(bf16_lo((uint32_t)x[e]), bf16_lo((uint32_t)y[e]), d);
        d = __builtin_fmaf(bf16_hi((uint32_t)x[e]), bf16_hi((uint32_t)y[e]), d);
      }
    }
#pragma unroll
    for (int m = 1; m < 8; m <<= 1) d += __shfl_xor(d, m, 64);
    if (c == 0) {
      // (a finite one stays finite in base 2, where a score that overflows with it is then -inf or +inf over it and not NaN: P = 0 or 1)
      const float l2 = l * ATTN_RCP_LN2, most = 0x1.fffffep127f;
      a.q_records[tile].lse2[r] = none ? __builtin_inff() : (__builtin_fabsf(l) <= most ? __builtin_amdgcn_fmed3f(l2, -most, most) : l2);
      a.q_records[tile].minus_d[r] = none ? 0.0f : -d;
    }
    __syncthreads();
    for (int k = tid; k < 4 * a.Dv; k += 256) a.g_rows[tile * 4 * a.Dv + k] = grad[k];
    return;
  }
  tile -= a.q_tiles;
  order_scales(a.ks, tile, a.D / 32, a.k_records[tile].scales);
  decode_tile(a.k, a.ks, tile, a.D, a.k_rows);
  const int lane = tid & 63, wave = tid >> 6, bands = a.Sk / 32;
  if (wave * 32 >= a.Dv) return;
  const int64_t bh = tile / bands, band = tile % bands;
  const uint8_t* column = a.vt + (bh * a.Dv + wave * 32 + (lane & 31)) * (int64_t)(a.Sk / 2) + band * 16 + 8 * (lane >> 5);
  const uint2 w = *reinterpret_cast<const uint2*>(column);   // 16 keys of one column
  const float scale = e8m0_value(a.vs[tile * (a.Dv / 32) + wave]);
  uint16_t* block = reinterpret_cast<uint16_t*>(turned[wave]);
  const v4i_t lo = decode8(w.x, scale), hi = decode8(w.y, scale);
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const uint32_t v = (uint32_t)(e < 4 ? lo[e & 3] : hi[e & 3]);
    const int key = 16 * (lane >> 5) + 2 * e;
    block[key * 40 + (lane & 31)] = (uint16_t)v;
    block[(key + 1) * 40 + (lane & 31)] = (uint16_t)(v >> 16);
  }
  wave_lds_order();
#pragma unroll
  for (int k = 0; k < 2; ++k) {   // the wave's four pieces of the 32 keys
    const int i = 64 * k + lane, p = i >> 5, key = (i & 31) ^ (p << 2);
    a.v_rows[tile * 4 * a.Dv + wave * 128 + i] = *reinterpret_cast<const v4i_t*>(turned[wave] + key * 20 + 4 * p);
  }
}

// Lists of tiles (see AttnBwdPlan) of one head: how many, of all together, the longest.
struct Lists {
  int64_t blocks, sum, longest;
};
void count_tiles(Lists& keys, Lists& rows, int64_t qn, int64_t kn, int causal) {
  const int64_t shift = kn - qn;
  auto add = [](Lists& l, int64_t n) {
    l.blocks += 1;
    l.sum += n;
    l.longest = n > l.longest ? n : l.longest;
  };
  for (int64_t at = 0; at < kn; at += BWD_BLOCK) {
    const int64_t first = causal && at > shift ? (at - shift) / 32 : 0;
    add(keys, first < qn / 32 ? qn / 32 - first : 0);
  }
  for (int64_t at = 0; at < qn; at += BWD_BLOCK) {
    const int64_t end = at + BWD_BLOCK < qn ? at + BWD_BLOCK : qn;
    add(rows, (causal ? end + shift : kn) / 32);
  }
}
// How long lists are cut.
struct Cuts {
  AttnBwdCut keys, rows;
  int rows_first;
};
AttnBwdCut cut_lists(bool cut, int64_t longest, int64_t piece, int most) {
  if (!cut) return {1, 1 << 30, nullptr};
  int64_t parts = (longest + piece - 1) / piece;
  if (parts > most) {
    parts = most;
    piece = (longest + most - 1) / most;
  }
  return {(int)parts, (int)(piece < (1 << 30) ? piece : 1 << 30), nullptr};
}
Cuts cut(const alto_mxfp4_attention_bwd_t& p) {
  const int64_t group = p.Hq / p.Hk;
  Lists keys{}, rows{};
  if (p.n_seqs > 0) {
    for (int i = 0; i < p.n_seqs; ++i) count_tiles(keys, rows, p.cu_q[i + 1] - p.cu_q[i], p.cu_k[i + 1] - p.cu_k[i], p.causal);
  } else {
    count_tiles(keys, rows, p.Sq, p.Sk_used, p.causal);
  }
  // Counted in tiles of dK and dV; one of dQ takes about .62 of one (products: 18 to 26 with D = Dv = 128).  The compute units hold 512 workgroups up to
  // D = 128 (above, 256; a share of 256 there was faster for one sequence of 192 / 64 on a few key heads, 238 -> 175 us, and slower for packed ones of 192,
  // 95 -> 117: 512 for all), and a list much longer than an equal share of the whole ends alone.  Pieces have 1.05 of that share (1.17 and 0.85: 3 % and 1.5 % more over 13 shapes) and
  // 24 tiles at least (16 and 32: 80.9 and 73.6 us for 72.2, 6 packed sequences of 16 / 4 heads of 128).  Parts cost a kernel, 5 tiles' time, and their
  // sums' way through memory.  So whichever of the two kinds is cut by what the launch would take: both, where few rows or heads leave all but some
  // units idle (3 x 6 / 3 heads, 64 rows, 4736 keys of 128 / 64: 32 us, 84 whole; 2048 tokens of 128, 4 heads 45, 57 whole), neither at 2048 tokens of
  // 20 heads (94 us, 102 with dK and dV cut) or 32 (124, 134), dK and dV at 12 (77, 82 whole) and 3 x 64 / 8 (655, 691 whole).
  const double B = (double)p.B, share = 1.05 * B * p.Hq * ((double)keys.sum + 0.62 * (double)rows.sum) / 512.0;
  const double key_piece = std::max(share, 24.0), row_piece = std::max(share / 0.62, 24.0);
  const double key_whole = (double)(keys.longest * group), row_whole = (double)rows.longest;
  const double key_cost = 0.042 * B * ((double)keys.sum * p.Hq / key_piece + (double)keys.blocks * p.Hk / 2) * (double)(p.D + p.Dv) / 256;
  const double row_cost = 0.04 * B * p.Hq * ((double)rows.sum / row_piece + (double)rows.blocks / 2) * (double)p.D / 128;
  bool best_keys = false, best_rows = false;
  double best = 0;
  for (int c = 0; c < 4; ++c) {
    const bool k = c & 1, r = c & 2;
    if ((k && key_whole <= 1.25 * key_piece) || (r && row_whole <= 1.25 * row_piece)) continue;
    const double time = std::max(share, std::max(k ? key_piece : key_whole, 0.62 * (r ? row_piece : row_whole))) + (c ? 5.0 : 0.0) + (k ? key_cost : 0.0) + (r ? row_cost : 0.0);
    if (c == 0 || time < best) {
      best = time;
      best_keys = k;
      best_rows = r;
    }
  }
  // The kind with the longer lists starts first: dQ's at 3 x 8 heads, 480 rows, 1056 keys of 192 / 128 with a bias (83 us, 89 last) or 4 x 16 heads, 256
  // rows, 4096 keys of 128 (161, 170); not where they are about as long (6 packed sequences of 16 / 4 heads of 64: 54, 50 last).
  const bool rows_first = 0.62 * (best_rows ? row_piece : row_whole) > 1.25 * (best_keys ? key_piece : key_whole);
  return {cut_lists(best_keys, keys.longest * group, (int64_t)key_piece, 16), cut_lists(best_rows, rows.longest, (int64_t)row_piece, 32), rows_first};
}

struct Workspace {
  int64_t q_records, k_records, k_rows, v_rows, g_rows, key_sums, row_sums, total;
};
Workspace workspace(const alto_mxfp4_attention_bwd_t& p, const Cuts& cuts) {
  const int64_t B = p.B, Hq = p.Hq, Hk = p.Hk, Sq = p.Sq, Sk = p.Sk, D = p.D, Dv = p.Dv;
  Workspace w{};
  int64_t at = 0;
  auto take = [&](int64_t& p, int64_t n) { p = at; at += (n + 255) / 256 * 256; };
  take(w.q_records, B * Hq * (Sq / 32) * (int64_t)sizeof(QRecord));
  take(w.k_records, B * Hk * (Sk / 32) * (int64_t)sizeof(KRecord));
  take(w.k_rows, B * Hk * Sk * D * 2);
  take(w.v_rows, B * Hk * Sk * Dv * 2);
  take(w.g_rows, B * Hq * Sq * Dv * 2);
  const int64_t more = p.n_seqs > 0 ? (p.n_seqs < ATTN_MAX_SEQS ? p.n_seqs : ATTN_MAX_SEQS) : 1;   // (blocks: at least those of any launch)
  take(w.key_sums, cuts.keys.parts > 1 ? B * Hk * (Sk / BWD_BLOCK + more) * cuts.keys.parts * BWD_BLOCK * (D + Dv) * 4 : 0);
  take(w.row_sums, cuts.rows.parts > 1 ? B * Hq * (Sq / BWD_BLOCK + more) * cuts.rows.parts * BWD_BLOCK * D * 4 : 0);
  w.total = at;
  return w;
}

int check_sizes(const alto_mxfp4_attention_bwd_t& p) {
  const long long B = p.B, Hq = p.Hq, Hk = p.Hk, Sq = p.Sq, Sk = p.Sk, D = p.D, Dv = p.Dv;
  ALTO_REQUIRE(B > 0 && Hq > 0 && Hk > 0 && Hq % Hk == 0, "attention_bwd: Hq=%lld must be a positive multiple of Hk=%lld", Hq, Hk);
  ALTO_REQUIRE(Sq > 0 && Sq % 32 == 0 && Sk > 0 && Sk % 32 == 0, "attention_bwd: Sq=%lld and Sk=%lld must be positive multiples of 32", Sq, Sk);
  ALTO_REQUIRE(D == 64 || D == 128 || D == 192 || D == 256, "attention_bwd: head dim D=%lld must be 64, 128, 192 or 256", D);
  ALTO_REQUIRE(Dv == 64 || Dv == 128, "attention_bwd: value dim Dv=%lld must be 64 or 128", Dv);
  ALTO_REQUIRE(B <= 65535 && Hq < (1ll << 31) && Sq <= 65535ll * 128 && Sk <= 65535ll * 128, "attention_bwd: B, Sq / 128 and Sk / 128 must stay below 65536");
  ALTO_REQUIRE(product_below(1ll << 40, B * Sq, Hq, D > Dv ? D : Dv) && product_below(1ll << 40, B * Sk, Hk, D > Dv ? D : Dv), "attention_bwd: tensor too large");
  // (a launch's threads, 256 a workgroup, are counted in 32 bits)
  ALTO_REQUIRE(B * Hq * (Sq / 32) + B * Hk * (Sk / 32) < (1ll << 24), "attention_bwd: tensor too large: 2^24 tiles of 32 rows or more");
  ALTO_REQUIRE(p.Sk_used > 0 && p.Sk_used <= p.Sk && p.Sk_used % 32 == 0, "attention_bwd: Sk_used=%lld must be a multiple of 32 in (0, Sk]", (long long)p.Sk_used);
  ALTO_REQUIRE(p.n_seqs >= 0, "attention_bwd: negative number of sequences");
  ALTO_REQUIRE(p.causal == 0 || p.n_seqs > 0 || p.Sq <= p.Sk_used, "attention_bwd: causal attention needs Sq <= Sk (got %lld > %lld)", (long long)p.Sq, (long long)p.Sk_used);
  if (p.n_seqs > 0) {
    ALTO_REQUIRE(p.cu_q && p.cu_k && p.B == 1 && p.Sk_used == p.Sk && !p.bias, "attention_bwd: packed sequences need their boundaries, B = 1, all keys used and no bias");
    ALTO_REQUIRE(p.cu_q[0] == 0 && p.cu_k[0] == 0 && p.cu_q[p.n_seqs] == p.Sq && p.cu_k[p.n_seqs] == p.Sk,
                 "attention_bwd: the sequence boundaries must run from 0 to the token counts");
    for (int i = 0; i < p.n_seqs; ++i) {
      ALTO_REQUIRE(p.cu_q[i + 1] > p.cu_q[i] && p.cu_k[i + 1] > p.cu_k[i] && p.cu_q[i + 1] % 32 == 0 && p.cu_k[i + 1] % 32 == 0,
                   "attention_bwd: sequence boundaries must be increasing multiples of 32 tokens");
      ALTO_REQUIRE(!p.causal || p.cu_q[i + 1] - p.cu_q[i] <= p.cu_k[i + 1] - p.cu_k[i], "attention_bwd: causal attention needs Sq <= Sk (got %d > %d)",
                   p.cu_q[i + 1] - p.cu_q[i], p.cu_k[i + 1] - p.cu_k[i]);
    }
  }
  return ALTO_MXFP4_OK;
}

}  // namespace

static int attention_bwd(const alto_mxfp4_attention_bwd_t& p, hipStream_t st) {
  if (const int rc = check_sizes(p)) return rc;
  ALTO_REQUIRE(p.q_codes && p.q_scales && p.k_codes && p.k_scales && p.vt_codes && p.v_scales && p.dout && p.out && p.lse && p.workspace && (p.dk || p.dq),
               "attention_bwd: null pointer");
  ALTO_REQUIRE(!p.dk == !p.dv, "attention_bwd: dk and dv are written together");
  ALTO_REQUIRE(((uintptr_t)p.q_codes | (uintptr_t)p.k_codes | (uintptr_t)p.dout | (uintptr_t)p.out | (uintptr_t)p.dq | (uintptr_t)p.dk | (uintptr_t)p.dv) % 16 == 0 &&
               (uintptr_t)p.vt_codes % 8 == 0, "attention_bwd: Q and K codes, dout, out and the gradients must be 16-byte aligned, V codes 8-byte aligned");
  ALTO_REQUIRE(((uintptr_t)p.lse | (uintptr_t)p.bias | (uintptr_t)p.alibi_slopes) % 4 == 0, "attention_bwd: lse, bias and slopes must be 4-byte aligned");
  for (const int64_t s : {p.dout_sb, p.dout_sh, p.dout_ss, p.out_sb, p.out_sh, p.out_ss, p.dq_sb, p.dq_sh, p.dq_ss, p.dk_sb, p.dk_sh, p.dk_ss, p.dv_sb, p.dv_sh, p.dv_ss})
    ALTO_REQUIRE(s >= 0 && s < (1ll << 40) && s % 8 == 0, "attention_bwd: strides of dout, out and the gradients must be non-negative multiples of 8 elements");
  for (const int64_t s : {p.lse_sb, p.lse_sh, p.lse_ss, p.bias_sb, p.bias_sh, p.bias_sm, p.alibi_sb, p.alibi_sh})
    ALTO_REQUIRE(s >= 0 && s < (1ll << 40), "attention_bwd: strides must be non-negative");
  ALTO_REQUIRE(p.sm_scale > 0.0f && p.sm_scale < __builtin_inff(), "attention_bwd: sm_scale must be positive and finite");
  ALTO_REQUIRE(p.sm_scale >= 0x1p-64f || (!p.bias && !p.alibi_slopes), "attention_bwd: sm_scale must be at least 2^-64 with a bias or slopes");
  ALTO_REQUIRE(!p.bias || p.bias_sm < (1 << 24), "attention_bwd: rows of the bias must be less than 2^24 elements apart");
  const Cuts cuts = cut(p);
  const Workspace w = workspace(p, cuts);
  ALTO_REQUIRE(p.workspace_bytes >= w.total && (uintptr_t)p.workspace % 256 == 0, "attention_bwd: the workspace must be 256-byte aligned and hold %lld bytes", (long long)w.total);
  std::unique_ptr<int[]> order;
  if (p.n_seqs > 0) {
    order.reset(new (std::nothrow) int[(size_t)p.n_seqs]);   // (no exception may leave a C entry)
    if (!order) {
      set_error("attention_bwd: no host memory for the order of %d sequences", p.n_seqs);
      return ALTO_MXFP4_ELAUNCH;
    }
  }
  uint8_t* ws = (uint8_t*)p.workspace;
  PrepareArgs r{};
  r.qs = (const uint8_t*)p.q_scales; r.k = (const uint8_t*)p.k_codes; r.ks = (const uint8_t*)p.k_scales;
  r.vt = (const uint8_t*)p.vt_codes; r.vs = (const uint8_t*)p.v_scales;
  r.dout = (const __bf16*)p.dout; r.out = (const __bf16*)p.out; r.lse = p.lse; r.alibi = p.alibi_slopes; r.alibi_sb = p.alibi_sb; r.alibi_sh = p.alibi_sh; r.sm_scale = p.sm_scale;
  r.do_sb = p.dout_sb; r.do_sh = p.dout_sh; r.do_ss = p.dout_ss; r.o_sb = p.out_sb; r.o_sh = p.out_sh; r.o_ss = p.out_ss;
  r.l_sb = p.lse_sb; r.l_sh = p.lse_sh; r.l_ss = p.lse_ss;
  r.Hq = (int)p.Hq; r.Hk = (int)p.Hk; r.Sq = (int)p.Sq; r.Sk = (int)p.Sk; r.D = (int)p.D; r.Dv = (int)p.Dv;
  r.q_tiles = (int)(p.B * p.Hq * (p.Sq / 32));
  r.q_records = (QRecord*)(ws + w.q_records); r.k_records = (KRecord*)(ws + w.k_records);
  r.k_rows = (v4i_t*)(ws + w.k_rows); r.v_rows = (v4i_t*)(ws + w.v_rows); r.g_rows = (v4i_t*)(ws + w.g_rows);
  hipLaunchKernelGGL(attn_bwd_prepare_kernel, dim3((unsigned)(r.q_tiles + (int)(p.B * p.Hk * (p.Sk / 32)))), dim3(256), 0, st, r);
  if (const int rc = check_launch("attention_bwd")) return rc;

  AttnBwdArgs a{};
  a.q = (const uint8_t*)p.q_codes; a.k = r.k; a.q_records = r.q_records; a.k_records = r.k_records;
  a.k_tiles = (const __bf16*)r.k_rows; a.v_tiles = (const __bf16*)r.v_rows; a.g_tiles = (const __bf16*)r.g_rows;
  a.dq = p.dq; a.dk = p.dk; a.dv = p.dv;
  a.dq_sb = p.dq_sb; a.dq_sh = p.dq_sh; a.dq_ss = p.dq_ss; a.dk_sb = p.dk_sb; a.dk_sh = p.dk_sh; a.dk_ss = p.dk_ss; a.dv_sb = p.dv_sb; a.dv_sh = p.dv_sh; a.dv_ss = p.dv_ss;
  a.B = (int)p.B; a.Hq = (int)p.Hq; a.Hk = (int)p.Hk; a.Sq = (int)p.Sq; a.Sk = (int)p.Sk; a.Sk_used = (int)p.Sk_used;
  a.sm_scale = p.sm_scale; a.causal = p.causal ? 1 : 0;
  a.bias = p.bias; a.bias_sb = p.bias_sb; a.bias_sh = p.bias_sh; a.bias_sm = p.bias_sm; a.distances = p.alibi_slopes != nullptr;
  const int row_block = BWD_BLOCK, key_block = row_block;
  auto go = [&](const AttnBwdSeqs& s, int q_blocks, int k_blocks) {
    AttnBwdPlan plan{q_blocks, k_blocks, cuts.keys, cuts.rows, 0, 0, cuts.rows_first, 0, 0};
    plan.keys.partial = (float*)(ws + w.key_sums);
    plan.rows.partial = (float*)(ws + w.row_sums);
    const int64_t key_blocks = p.dk ? p.B * p.Hk * k_blocks : 0, row_blocks = p.dq ? p.B * p.Hq * q_blocks : 0;
    const int64_t key_groups = (key_blocks * cuts.keys.parts + 7) / 8 * 8, row_groups = (row_blocks * cuts.rows.parts + 7) / 8 * 8;
    const int64_t key_sums = cuts.keys.parts > 1 ? key_blocks : 0, row_sums = cuts.rows.parts > 1 ? row_blocks : 0;
    ALTO_REQUIRE(key_groups + row_groups < (1ll << 24) && (key_sums + row_sums) * 12 < (1ll << 24), "attention_bwd: too many workgroups");
    plan.key_groups = (int)key_groups;
    plan.row_groups = (int)row_groups;
    plan.key_sums = (int)key_sums;
    plan.row_sums = (int)row_sums;
    switch (p.D) {
      case 64: return launch_attn_bwd<1>(a, s, plan, p.Dv, st);
      case 128: return launch_attn_bwd<2>(a, s, plan, p.Dv, st);
      case 192: return launch_attn_bwd<3>(a, s, plan, p.Dv, st);
      default: return launch_attn_bwd<4>(a, s, plan, p.Dv, st);
    }
  };
  AttnBwdSeqs s;
  s.n = 0;
  s.zq[0] = s.zk[0] = 0;
  if (p.n_seqs == 0) return go(s, (int)((p.Sq + row_block - 1) / row_block), (int)((p.Sk + key_block - 1) / key_block));
  for (int i = 0; i < p.n_seqs; ++i) order[(size_t)i] = i;
  std::sort(order.get(), order.get() + p.n_seqs, [&](int x, int y) {   // longest first
    const int kx = p.cu_k[x + 1] - p.cu_k[x], ky = p.cu_k[y + 1] - p.cu_k[y];
    return kx != ky ? kx > ky : x < y;
  });
  for (int at = 0; at < p.n_seqs;) {
    s.n = 0;
    for (; at < p.n_seqs && s.n < ATTN_MAX_SEQS; ++at) {
      const int i = order[(size_t)at], n = s.n, qn = p.cu_q[i + 1] - p.cu_q[i], kn = p.cu_k[i + 1] - p.cu_k[i];
      s.q0[n] = p.cu_q[i]; s.qn[n] = qn; s.k0[n] = p.cu_k[i]; s.kn[n] = kn;
      s.zq[n + 1] = s.zq[n] + (qn + row_block - 1) / row_block;
      s.zk[n + 1] = s.zk[n] + (kn + key_block - 1) / key_block;
      ++s.n;
    }
    if (const int rc = go(s, s.zq[s.n], s.zk[s.n])) return rc;
  }
  return ALTO_MXFP4_OK;
}

}  // namespace alto

extern "C" int64_t alto_mxfp4_attention_bwd_workspace_bytes(const alto_mxfp4_attention_bwd_t* p) {
  if (!p) {
    alto::set_error("attention_bwd_workspace_bytes: null pointer");
    return ALTO_MXFP4_EINVAL;
  }
  if (const int rc = alto::check_sizes(*p)) return rc;
  return alto::workspace(*p, alto::cut(*p)).total;
}

extern "C" int alto_mxfp4_attention_bwd(const alto_mxfp4_attention_bwd_t* p, void* stream) {
  ALTO_REQUIRE(p, "attention_bwd: null pointer");
  return alto::attention_bwd(*p, (hipStream_t)stream);
}
