// What the files of the attention backward share (attention_backward.hip: preparation and entry points; attention_backward_*.hip: the
// kernels of one head dim).
#pragma once
#include "attention.h"

namespace alto {

// Operands of the gradient kernel.  "Tile": 32 rows of a head; the preparation kernel writes what comes from the workspace, tile after tile.
struct AttnBwdArgs {
  const uint8_t* q;             // codes [B, Hq, Sq, D/2]
  const uint8_t* k;             // codes [B, Hk, Sk, D/2]
  const uint8_t* q_scales;      // workspace: 8 bytes a tile, that of columns 64 s + 32 h .. + 32 at 4 h + s
  const uint8_t* k_scales;
  const __bf16 *q_tiles, *k_tiles, *v_tiles, *g_tiles;   // workspace: bf16 tiles (RowTile) of Q, K, V as their codes have them, and of dO
  const float* stats;           // workspace: of every tile of Q, 32 times lse log2(e) (+inf for a row that sees no key), then 32 times -dO . O
  void *dq, *dk, *dv;           // bf16, element (b, h, row, column) at these strides, unit stride along the head dim; dq, or dk and dv, may be NULL: not wanted
  int64_t dq_sb, dq_sh, dq_ss, dk_sb, dk_sh, dk_ss, dv_sb, dv_sh, dv_ss;
  int B, Hq, Hk, Sq, Sk, Sk_used;
  float sm_scale;
  int causal;
  const float* bias;  int64_t bias_sb, bias_sh, bias_sm;
  const float* alibi; int64_t alibi_sb, alibi_sh;
};

// Where 16-byte piece `p` of row `row` (columns 8 p .. 8 p + 7) sits in a tile of bf16 rows: the 32 rows' pieces of the same columns side by side,
// the rows in groups of four that change places from piece to piece.  Two kinds of read take a tile apart: fragments along the columns (16
// consecutive rows at one piece) and transposed ones (4 rows x 64 bytes); either meets all banks of the LDS once, and all of a tile's
// fragments sit at constant distances from one or two addresses a lane.
__host__ __device__ __forceinline__ constexpr int tile_piece(int row, int p) { return p * 32 + (row ^ ((p & 3) << 2)); }

// Sequences as AttnSeqs has them, the blocks of queries (dQ) and of keys (dK, dV) of sequence i at zq[i] and zk[i]; n = 0: B sequences of one length.
struct AttnBwdSeqs {
  int n;
  int zq[ATTN_MAX_SEQS + 1], zk[ATTN_MAX_SEQS + 1], q0[ATTN_MAX_SEQS], qn[ATTN_MAX_SEQS], k0[ATTN_MAX_SEQS], kn[ATTN_MAX_SEQS];
};

// How a launch is cut into workgroups: first those of dK, then those of dV, then those of dQ.  A block of keys walks the tiles of 32 rows that see
// it, of all query heads on its key head; lists longer than `chunk` are dealt out to up to `parts` workgroups, whose fp32 sums meet in a
// kernel of their own (`partial`: one set of accumulators for each gradient, part and block).
struct AttnBwdPlan {
  int q_blocks, k_blocks;       // over all sequences
  int parts, chunk;
  int key_groups, row_groups;   // workgroups of dK (and as many of dV; a multiple of 8), of dQ
  float* partial;
};
constexpr int ATTN_BWD_BLOCK = 128;   // keys or query rows of a workgroup

template <int NK>
int launch_attn_bwd(const AttnBwdArgs& a, const AttnBwdSeqs& seqs, const AttnBwdPlan& plan, int64_t Dv, hipStream_t st);

#ifdef ALTO_ATTENTION_BACKWARD_KERNELS
namespace {

typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef short v4s_t __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) uint8_t lds_u8;
typedef __attribute__((address_space(3))) v4s_t lds_v4s;

// A tile of 32 rows of bf16, W columns, in the LDS
template <int W>
struct RowTile {
  static constexpr int BYTES = 32 * W * 2;
  // lane (r, h)'s columns 16 i + 8 h .. + 8 of row r: the swizzle of piece 2 i + h depends on i's lowest bit
  __device__ static __forceinline__ int row_base(int lane, int odd) { return tile_piece(lane & 31, 2 * odd + (lane >> 5)) * 16 - odd * 1024; }
  __device__ static __forceinline__ bf16x8_t row_frag(const uint8_t* at, int i) { return *reinterpret_cast<const bf16x8_t*>(at + i * 1024); }
  // lane (r, h)'s column 32 n + r of the rows 16 c + 4 h + 0..3 and 16 c + 8 + 4 h + 0..3: the order in which a score tile's registers
  // 8 c .. 8 c + 7 hold its rows.  A transposed read hands lane i of 16 the column i of four rows that the 16 lanes fetch 8 bytes each of.
  __device__ static __forceinline__ int column_base(int lane, int upper) {
    const int j = lane & 15, g = (lane >> 4) & 1, h = lane >> 5;
    return tile_piece(8 * upper + 4 * h + (j >> 2), 2 * g + ((j & 3) >> 1)) * 16 + 8 * (j & 1);
  }
  __device__ static __forceinline__ bf16x8_t column_frag(const uint8_t* lower, const uint8_t* upper, int n, int c) {
    const int at = n * 2048 + c * 256;
    const v4s_t lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s*)(const __attribute__((address_space(3))) void*)(lower + at));
    const v4s_t hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s*)(const __attribute__((address_space(3))) void*)(upper + at));
    return __builtin_bit_cast(bf16x8_t, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
  }
};

// 32 rows of codes, D/2 bytes each, in the LDS: the rows' 16-byte pieces of the same columns side by side
template <int NK>
struct CodeTile {
  static constexpr int D = NK * 64, BYTES = 32 * (D / 2);
  __device__ static __forceinline__ int source(int i) { return (i & 31) * (D / 2) + (i >> 5) * 16; }   // of piece i of the tile
};

__device__ __forceinline__ __amdgpu_buffer_rsrc_t buffer(const void* p, int64_t bytes) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(p), 0, (int)bytes, 0x00020000);
}
__device__ __forceinline__ void load_piece(__amdgpu_buffer_rsrc_t src, const uint8_t* to, int lane_offset, int offset) {   // (`offset` the same in all lanes)
  __builtin_amdgcn_raw_ptr_buffer_load_lds(src, (__attribute__((address_space(3))) void*)to, 16, lane_offset, offset, 0, 0);
}

// score register v of half h <-> row 8 (v / 4) + 4 h + v % 4 of the tile
__device__ __forceinline__ int score_row(int v, int h) { return 8 * (v >> 2) + 4 * h + (v & 3); }

// lane (r, h) stores row r of a transposed accumulator (registers: columns 32 n + score_row(v, h)) as bf16
__device__ __forceinline__ void store_columns(__bf16* row, const v16f_t& acc, float scale, int n, int h) {
#pragma unroll
  for (int g = 0; g < 4; ++g) {
    const uint2 w = make_uint2(pack_bf16x2(acc[4 * g] * scale, acc[4 * g + 1] * scale), pack_bf16x2(acc[4 * g + 2] * scale, acc[4 * g + 3] * scale));
    *reinterpret_cast<uint2*>(row + 32 * n + 8 * g + 4 * h) = w;
  }
}

__device__ __forceinline__ v16f_t zeros() {
  v16f_t z;
#pragma unroll
  for (int v = 0; v < 16; ++v) z[v] = 0.0f;
  return z;
}

struct AttnBwdBlock {
  int qn, kn, q_first, k_first, block;
};
template <bool KEYS>
__device__ __forceinline__ AttnBwdBlock attn_bwd_block(const AttnBwdArgs& a, const AttnBwdSeqs& s, int z) {
  AttnBwdBlock w{a.Sq, a.Sk_used, 0, 0, z};
  if (s.n) {
    const int* z0 = KEYS ? s.zk : s.zq;
    int lo = 0, hi = s.n - 1;
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (z0[mid] <= z) lo = mid; else hi = mid - 1;
    }
    w = AttnBwdBlock{s.qn[lo], s.kn[lo], s.q0[lo], s.k0[lo], z - z0[lo]};
  }
  return w;
}

// Eight neighbouring workgroups go to the eight XCDs in turn: each XCD gets a range of consecutive (batch, head) pairs, so that a head's
// operands come into one L2.
__device__ __forceinline__ int head_of(int i, int heads) { return heads % 8 == 0 ? (i & 7) * (heads >> 3) + (i >> 3) : i; }

// The list of a block of keys: tiles first .. all of each of the group's heads.
struct KeyList {
  int first, each, total, parts;
};
__device__ __forceinline__ KeyList key_list(const AttnBwdArgs& a, const AttnBwdBlock& w, const AttnBwdPlan& plan) {
  KeyList l{0, 0, 0, 1};
  const int all = w.qn / 32;
  if (a.causal) {
    l.first = (w.block * ATTN_BWD_BLOCK - (w.kn - w.qn)) / 32;
    l.first = l.first < 0 ? 0 : l.first;
  }
  l.each = l.first < all && w.block * ATTN_BWD_BLOCK < w.kn ? all - l.first : 0;
  l.total = l.each * (a.Hq / a.Hk);
  l.parts = (l.total + plan.chunk - 1) / plan.chunk;
  l.parts = l.parts < 1 ? 1 : (l.parts > plan.parts ? plan.parts : l.parts);
  return l;
}

// The three gradients have one shape.  A wave holds 32 rows (of K for dK and dV, of Q for dQ: "its own side") and walks tiles of 32 rows of the
// other side, from which it takes
//   the codes, for the scores        S = codes x own codes                 (rows of the tile in registers, its own in lanes),
//   bf16 rows, for dP                V or dO x own dO or V                 (dK, dQ),
//   bf16 rows by columns, the factor of its sums   dK += dS^T Q, dQ += dS K, dV += P^T dO.
enum AttnBwdKind { BWD_DQ, BWD_DK, BWD_DV };

template <int KIND, int NK, int NV>
struct BwdTile {
  static constexpr int NA = KIND == BWD_DV ? NV : NK;   // width of the gradient / 64
  static constexpr int CODES = CodeTile<NK>::BYTES, INNER = KIND == BWD_DV ? 0 : RowTile<64 * NV>::BYTES, FACTOR = RowTile<64 * NA>::BYTES;
  // three slots of each, four of the statistics
  static constexpr int O_INNER = 3 * CODES, O_FACTOR = O_INNER + 3 * INNER, O_STATS = O_FACTOR + 3 * FACTOR, LDS = O_STATS + (KIND == BWD_DQ ? 0 : 4 * 256);
  static constexpr int SCORE_LOADS = 1 + (KIND != BWD_DQ && NK == 4 ? 1 : 0) + (KIND == BWD_DV ? 0 : NV), LOADS = SCORE_LOADS + NA;   // of a wave, each step
  static constexpr int64_t PARTIAL = (int64_t)4 * 2 * NA * 16 * 64;   // floats of a workgroup's sums

  // The products of a step, in order: those of the scores, then by turns one of dP and one of the sums.
  static constexpr int NS = NK, NI = KIND == BWD_DV ? 0 : 4 * NV, NF = 4 * NA, PRODUCTS = NS + NI + NF;
  struct Op {
    int kind, j;   // 0: S, 1: dP, 2: sums
  };
  static constexpr Op op(int i) {
    if (i < NS) return {0, i};
    int inner = 0, factor = 0;
    for (int k = NS;; ++k) {
      const bool take_inner = inner < NI && (factor == NF || inner * NF <= factor * NI);
      if (k == i) return take_inner ? Op{1, inner} : Op{2, factor};
      if (take_inner) ++inner; else ++factor;
    }
  }
};

template <int KIND, int NK, int NV, bool BIASED>
__device__ __forceinline__ void attn_bwd_body(const AttnBwdArgs& a, const AttnBwdSeqs& seqs, const AttnBwdPlan& plan, int item, __bf16* __restrict__ grad_out,
                                              float* __restrict__ partial, uint8_t* lds) {
  using T = BwdTile<KIND, NK, NV>;
  using IT = RowTile<64 * NV>;
  using FT = RowTile<64 * T::NA>;
  constexpr bool KEYS = KIND != BWD_DQ;
  constexpr int D = 64 * NK, DV = 64 * NV, NA = T::NA;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), r = lane & 31, h = lane >> 5;

  // ---- what this workgroup works on
  const int heads = a.B * (KEYS ? a.Hk : a.Hq), bh = head_of(item % heads, heads), group = a.Hq / a.Hk;
  const int part = KEYS ? (item / heads) % plan.parts : 0;
  int z = KEYS ? item / heads / plan.parts : item / heads;
  if (KEYS && z >= plan.k_blocks) return;
  if (!KEYS && a.causal && !seqs.n) z = plan.q_blocks - 1 - z;
  const AttnBwdBlock w = attn_bwd_block<KEYS>(a, seqs, z);
  const int b = bh / (KEYS ? a.Hk : a.Hq), head = bh % (KEYS ? a.Hk : a.Hq);
  const int shift = w.kn - w.qn, own0 = w.block * ATTN_BWD_BLOCK + wave * 32;   // the wave's first row in its sequence
  const bool live = own0 < (KEYS ? w.kn : w.qn);
  int first = 0, last, begin = 0, total, parts = 1;   // the other side's tiles first .. last (of each head), and this workgroup's part of the list
  if constexpr (KEYS) {
    const KeyList list = key_list(a, w, plan);
    if (part >= list.parts) return;
    parts = list.parts;
    first = list.first;
    last = w.qn / 32;
    begin = (int)((int64_t)list.total * part / parts);
    total = (int)((int64_t)list.total * (part + 1) / parts) - begin;
  } else {
    last = w.kn / 32;
    if (a.causal) {
      const int end = (w.block + 1) * ATTN_BWD_BLOCK < w.qn ? (w.block + 1) * ATTN_BWD_BLOCK : w.qn;
      last = (end + shift) / 32;
    }
    total = last;
  }
  const int own_tile = (KEYS ? bh * (a.Sk / 32) + w.k_first / 32 : bh * (a.Sq / 32) + w.q_first / 32) + (live ? own0 / 32 : 0);   // among all tiles of its side

  v16f_t acc[2 * NA];
#pragma unroll
  for (int n = 0; n < 2 * NA; ++n) acc[n] = zeros();

  if (total > 0) {
    // ---- its own side, in registers
    v8i_t xf[NK];
    bf16x8_t yf[KIND == BWD_DV ? 1 : 4 * NV];
    float lse2 = 0.0f;
    v16f_t nd;
#pragma unroll
    for (int s = 0; s < NK; ++s) xf[s] = frag16((KEYS ? a.k : a.q) + ((int64_t)own_tile * 32 + r) * (D / 2) + s * 32 + h * 16);
    const uint32_t x_scales = *reinterpret_cast<const uint32_t*>((KEYS ? a.k_scales : a.q_scales) + (int64_t)own_tile * 8 + 4 * h);
    if constexpr (KIND != BWD_DV) {
      const uint8_t* y = reinterpret_cast<const uint8_t*>(KEYS ? a.v_tiles : a.g_tiles) + (int64_t)own_tile * IT::BYTES;
#pragma unroll
      for (int i = 0; i < 4 * NV; ++i) yf[i] = IT::row_frag(y + IT::row_base(lane, i & 1), i);
    }
    if constexpr (!KEYS) {
      lse2 = a.stats[(int64_t)own_tile * 64 + r];
      const float x = a.stats[(int64_t)own_tile * 64 + 32 + r];
#pragma unroll
      for (int v = 0; v < 16; ++v) nd[v] = x;
    }

    // ---- the other side's tiles
    struct Place {
      int tile, at;   // in its sequence, among all
    };
    const int tiles = KEYS ? a.Sq / 32 : a.Sk / 32;   // of a head
    int next_tile = first, left = total, next_base = KEYS ? (b * a.Hq + head * group) * tiles + w.q_first / 32 : (b * a.Hk + head / group) * tiles + w.k_first / 32;
    if (KEYS && begin > 0) {
      next_base += begin / (last - first) * tiles;
      next_tile += begin % (last - first);
    }
    auto next = [&]() {   // (past the end: the last tile again)
      const Place p{next_tile, next_base + next_tile};
      if (--left > 0 && ++next_tile == last) {
        next_tile = first;
        next_base += tiles;
      }
      return p;
    };
    const int o_codes = CodeTile<NK>::source(64 * (wave % NK) + lane), o_linear = wave * 1024 + lane * 16;
    const uint8_t* const codes = KEYS ? a.q : a.k;
    const uint8_t* const inner = reinterpret_cast<const uint8_t*>(KEYS ? a.g_tiles : a.v_tiles);
    const uint8_t* const factor = reinterpret_cast<const uint8_t*>(KIND == BWD_DV ? a.g_tiles : (KEYS ? a.q_tiles : a.k_tiles));
    const uint8_t* const scales = (KEYS ? a.q_scales : a.k_scales) + 4 * h;
    auto load_scores = [&](const Place& p, int slot, int t) {   // what S and dP need, and the statistics
      if (!KEYS || NK == 4 || wave < NK) load_piece(buffer(codes + (int64_t)p.at * T::CODES, T::CODES), lds + slot * T::CODES + 1024 * (wave % NK), o_codes, 0);   // (dQ: waves past the last piece repeat one)
      if constexpr (KEYS) {
        if (NK == 4 || wave >= NK)
          __builtin_amdgcn_raw_ptr_buffer_load_lds(buffer(a.stats + (int64_t)p.at * 64, 256), (__attribute__((address_space(3))) void*)(lds + T::O_STATS + (t & 3) * 256), 4, lane * 4, 0, 0, 0);
      }
      if constexpr (KIND != BWD_DV) {
        const __amdgpu_buffer_rsrc_t from = buffer(inner + (int64_t)p.at * T::INNER, T::INNER);
#pragma unroll
        for (int j = 0; j < NV; ++j) load_piece(from, lds + T::O_INNER + slot * T::INNER + 1024 * (4 * j + wave), o_linear, 4096 * j);
      }
    };
    auto load_factor = [&](const Place& p, int slot) {
      const __amdgpu_buffer_rsrc_t from = buffer(factor + (int64_t)p.at * T::FACTOR, T::FACTOR);
#pragma unroll
      for (int j = 0; j < NA; ++j) load_piece(from, lds + T::O_FACTOR + slot * T::FACTOR + 1024 * (4 * j + wave), o_linear, 4096 * j);
    };
    auto scales_of = [&](const Place& p) { return *reinterpret_cast<const uint32_t*>(scales + (int64_t)p.at * 8); };
    auto wait_all_but = [](auto n) { __builtin_amdgcn_s_waitcnt(0x0070 | 0x0F00 | (decltype(n)::value & 15)); };

    const int code_base = lane * 16, row_base[2] = {IT::row_base(lane, 0), IT::row_base(lane, 1)}, column_base[2] = {FT::column_base(lane, 0), FT::column_base(lane, 1)};
    const float c2 = a.sm_scale * ATTN_RCP_LN2;

    // Which rows of the tile the lane sees, in the bits of the packed pairs: most tiles are seen whole (state 2), the diagonal's in part (1), a tile
    // before its diagonal not at all (0: another wave of the workgroup needs it).
    uint32_t seen[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) seen[i] = ~0u;
    int state = 2;
    auto look = [&](const Place& p) {
      if (!a.causal) return;
      const int away = KEYS ? 32 * p.tile + shift - own0 : own0 + shift - 32 * p.tile;   // a multiple of 32
      const int now = away > 0 ? 2 : (away == 0 ? 1 : 0);
      if (now == state) return;
      state = now;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int x = score_row(2 * i, h);   // the pair's first row; the second is the next one
        const bool lo = KEYS ? x >= r : x <= r, hi = KEYS ? x + 1 >= r : x + 1 <= r;
        seen[i] = now == 2 ? ~0u : (now == 1 ? (lo ? 0xFFFFu : 0u) | (hi ? 0xFFFF0000u : 0u) : 0u);
      }
    };

    // ---- Three stages in one step: S and dP of tile t + 1 and the sums' product with tile t - 1 on the matrix pipe, the probabilities of tile t
    // on the vector pipe.  Loads go out two steps before they are used: a step starts those of the scores of t + 3 and the factor of t + 1, and
    // ends with a wait for everything that earlier steps started.  The products are issued in a fixed order (sched_barrier): the read of
    // an operand AHEAD products before its use, a sixteenth of the vector work behind each.  Left to itself the compiler puts every read right
    // in front of its product and waits there.
    constexpr int AHEAD = 4, HALVES = 16;
    struct Scores {
      v16f_t S, dp;
    };
    // (RUN: the first step only has scores to compute)
    auto step = [&](auto run, int t, int slot, const Place& p, uint32_t sc, const Scores& from, const bf16x8_t (&f)[2], Scores& to, bf16x8_t (&f_next)[2]) {
      constexpr bool RUN = decltype(run)::value;
      const int after = slot == 2 ? 0 : slot + 1, before = slot == 0 ? 2 : slot - 1;
      const uint8_t* const at_codes = lds + after * T::CODES + code_base;
      const uint8_t* at_rows[2];
      const uint8_t* at_columns[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        at_rows[i] = lds + T::O_INNER + after * T::INNER + row_base[i];
        at_columns[i] = lds + T::O_FACTOR + before * T::FACTOR + column_base[i];
      }
      const float* const stats = reinterpret_cast<const float*>(lds + T::O_STATS + (t & 3) * 256) + 4 * h;
      const float* const stats_next = reinterpret_cast<const float*>(lds + T::O_STATS + ((t + 1) & 3) * 256) + 4 * h;
      constexpr int N = RUN ? T::PRODUCTS : T::NS + T::NI;
      auto op = [](int i) constexpr { return RUN ? T::op(i) : typename T::Op{i < T::NS ? 0 : 1, i < T::NS ? i : i - T::NS}; };
      bf16x8_t frag[AHEAD + 1];
      auto read = [&](auto ic) {
        constexpr int i = decltype(ic)::value;
        if constexpr (i < N) {
          constexpr typename T::Op o = op(i);
          bf16x8_t& x = frag[i % (AHEAD + 1)];
          if constexpr (o.kind == 0) x = *reinterpret_cast<const bf16x8_t*>(at_codes + o.j * 1024);
          else if constexpr (o.kind == 1) x = IT::row_frag(at_rows[o.j & 1], o.j);
          else x = FT::column_frag(at_columns[0], at_columns[1], o.j % (2 * NA), o.j / (2 * NA));
        }
      };
      auto product = [&](auto ic) {
        constexpr int i = decltype(ic)::value;
        constexpr typename T::Op o = op(i);
        const bf16x8_t& x = frag[i % (AHEAD + 1)];
        if constexpr (o.kind == 0) {
          const v4i_t q = __builtin_bit_cast(v4i_t, x);
          to.S = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(v8i_t{q[0], q[1], q[2], q[3], 0, 0, 0, 0}, xf[o.j], o.j == 0 ? zeros() : to.S, 4, 4, o.j, (int)sc, o.j, (int)x_scales);
        } else if constexpr (o.kind == 1) {
          if constexpr (!KEYS && o.j == 0) to.dp = __builtin_amdgcn_mfma_f32_32x32x16_bf16(x, yf[o.j], nd, 0, 0, 0);
          else to.dp = __builtin_amdgcn_mfma_f32_32x32x16_bf16(x, yf[o.j], to.dp, 0, 0, 0);
        } else {
          acc[o.j % (2 * NA)] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(x, f[o.j / (2 * NA)], acc[o.j % (2 * NA)], 0, 0, 0);
        }
      };
      // P or dS of tile t, a pair of rows at a time, in two halves
      v4f_t l4[2];
      float e[8][2];
      uint32_t out[8];
      auto read_stats = [&](int g) {
        if constexpr (KEYS) l4[g & 1] = *reinterpret_cast<const v4f_t*>(stats + 8 * g);
      };
      auto half = [&](auto uc) {
        constexpr int u = decltype(uc)::value, i = u >> 1;
        if constexpr ((u & 1) == 0) {
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            const int v = 2 * i + k;
            float y = __builtin_fmaf(from.S[v], c2, -(KEYS ? l4[(v >> 2) & 1][v & 3] : lse2));
            if constexpr (BIASED) {
              const int there = 32 * p.tile + score_row(v, h), here = live ? own0 + r : 0;
              const int row = KEYS ? there : here, key = KEYS ? here : there;
              const int64_t hq = KEYS ? p.at / tiles - b * a.Hq : head;
              if (a.bias) y = __builtin_fmaf(a.bias[b * a.bias_sb + hq * a.bias_sh + row * a.bias_sm + key], ATTN_RCP_LN2, y);
              if (a.alibi) y = __builtin_fmaf(-a.alibi[b * a.alibi_sb + hq * a.alibi_sh] * ATTN_RCP_LN2, __builtin_fabsf((float)(row + shift - key)), y);
            }
            e[i][k] = __builtin_amdgcn_exp2f(y);
          }
          if constexpr (KEYS && (i & 1) == 1 && i / 2 + 2 < 4) read_stats(i / 2 + 2);   // (the group's last use is behind us)
        } else {
          if constexpr (KIND != BWD_DV) {
            e[i][0] *= from.dp[2 * i];
            e[i][1] *= from.dp[2 * i + 1];
          }
          out[i] = pack_bf16x2(e[i][0], e[i][1]) & seen[i];
          asm volatile("" : "+v"(out[i]));   // (here: otherwise it is moved behind the step, to where it is used)
        }
      };
      __builtin_amdgcn_sched_barrier(0);
      if constexpr (RUN) {
        read_stats(0);
        read_stats(1);
      }
      if constexpr (KIND == BWD_DK) {
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const v4f_t x = *reinterpret_cast<const v4f_t*>(stats_next + 32 + 8 * g);
#pragma unroll
          for (int i = 0; i < 4; ++i) to.dp[4 * g + i] = x[i];
        }
      }
      static_for<AHEAD>([&](auto ic) { read(ic); });
      __builtin_amdgcn_sched_barrier(0);
      static_for<N>([&](auto ic) {
        constexpr int i = decltype(ic)::value;
        read(std::integral_constant<int, i + AHEAD>{});
        product(ic);
        if constexpr (RUN) {
          constexpr int u0 = HALVES * i / N, u1 = HALVES * (i + 1) / N;
          static_for<u1 - u0>([&](auto uc) { half(std::integral_constant<int, u0 + decltype(uc)::value>{}); });
        }
        __builtin_amdgcn_sched_barrier(0);
      });
      if constexpr (RUN) {
#pragma unroll
        for (int c = 0; c < 2; ++c) f_next[c] = __builtin_bit_cast(bf16x8_t, v4i_t{(int)out[4 * c], (int)out[4 * c + 1], (int)out[4 * c + 2], (int)out[4 * c + 3]});
      }
    };

    Place p0 = next();
    load_scores(p0, 0, 0);
    load_factor(p0, 0);
    load_factor(p0, 2);   // (what the first step multiplies with zeros)
    Place p1 = next();
    load_scores(p1, 1, 1);
    Place p2 = next();
    uint32_t sc = scales_of(p0), sc1 = scales_of(p1);
    load_scores(p2, 2, 2);
    wait_all_but(std::integral_constant<int, T::SCORE_LOADS>{});
    asm volatile("s_barrier" ::: "memory");
    Scores x, y;
    bf16x8_t f[2], g[2];
    f[0] = f[1] = __builtin_bit_cast(bf16x8_t, v4i_t{0, 0, 0, 0});
    step(std::false_type{}, -1, 2, p0, sc, x, f, x, f);
    int slot = 0;   // of tile t
    auto whole_step = [&](int t, const Scores& from, const bf16x8_t (&f_now)[2], Scores& to, bf16x8_t (&f_next)[2]) {
      const int after = slot == 2 ? 0 : slot + 1;
      sc = sc1;
      sc1 = scales_of(p2);
      const Place p3 = next();
      load_scores(p3, slot, t + 3);
      load_factor(p1, after);
      look(p0);
      step(std::true_type{}, t, slot, p0, sc, from, f_now, to, f_next);
      p0 = p1;
      p1 = p2;
      p2 = p3;
      slot = after;
      wait_all_but(std::integral_constant<int, T::LOADS>{});
      asm volatile("s_barrier" ::: "memory");
    };
    auto final_sums = [&](const bf16x8_t (&f_now)[2]) {
      const uint8_t* at = lds + T::O_FACTOR + (slot == 0 ? 2 : slot - 1) * T::FACTOR;
#pragma unroll
      for (int c = 0; c < 2; ++c)
#pragma unroll
        for (int n = 0; n < 2 * NA; ++n) acc[n] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(FT::column_frag(at + column_base[0], at + column_base[1], n, c), f_now[c], acc[n], 0, 0, 0);
    };
    int t = 0;
    for (; t + 1 < total; t += 2) {
      whole_step(t, x, f, y, g);
      whole_step(t + 1, y, g, x, f);
    }
    if (t < total) {
      whole_step(t, x, f, y, g);
      f[0] = g[0];
      f[1] = g[1];
    }
    final_sums(f);
    wait_all_but(std::integral_constant<int, 0>{});   // (the last loads into the LDS, which nobody reads, before it is given back)
  }

  // ---- results
  if (KEYS && parts > 1) {
    v4f_t* to = reinterpret_cast<v4f_t*>(partial + (((int64_t)z * plan.parts + part) * heads + bh) * T::PARTIAL) + wave * (2 * NA * 4 * 64) + lane;
#pragma unroll
    for (int n = 0; n < 2 * NA; ++n)
#pragma unroll
      for (int g = 0; g < 4; ++g) to[(n * 4 + g) * 64] = v4f_t{acc[n][4 * g], acc[n][4 * g + 1], acc[n][4 * g + 2], acc[n][4 * g + 3]};
    return;
  }
  if (own0 >= (KEYS ? (seqs.n ? w.kn : a.Sk) : w.qn)) return;
  const int64_t sb = KIND == BWD_DQ ? a.dq_sb : (KIND == BWD_DK ? a.dk_sb : a.dv_sb), sh = KIND == BWD_DQ ? a.dq_sh : (KIND == BWD_DK ? a.dk_sh : a.dv_sh),
                ss = KIND == BWD_DQ ? a.dq_ss : (KIND == BWD_DK ? a.dk_ss : a.dv_ss);
  __bf16* row = grad_out + b * sb + head * sh + (int64_t)((KEYS ? w.k_first : w.q_first) + own0 + r) * ss;
#pragma unroll
  for (int n = 0; n < 2 * NA; ++n) store_columns(row, live ? acc[n] : zeros(), KIND == BWD_DV ? 1.0f : a.sm_scale, n, h);   // (keys behind the used ones: zeros)
}

// Sums of the parts, in their order.  Grid: (heads, key blocks, blocks of 32 columns of dK, then of dV).
template <int NK, int NV>
__global__ __launch_bounds__(256) void attn_bwd_sum_kernel(AttnBwdArgs a, AttnBwdSeqs seqs, AttnBwdPlan plan) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r = lane & 31, h = lane >> 5;
  const int heads = a.B * a.Hk, bh = blockIdx.x, z = blockIdx.y;
  const bool is_k = blockIdx.z < 2 * NK;
  const int n = is_k ? blockIdx.z : blockIdx.z - 2 * NK, width = is_k ? 2 * NK : 2 * NV;
  const AttnBwdBlock w = attn_bwd_block<true>(a, seqs, z);
  const KeyList list = key_list(a, w, plan);
  const int key = w.block * ATTN_BWD_BLOCK + wave * 32;
  if (list.parts == 1 || key >= (seqs.n ? w.kn : a.Sk)) return;
  const int hk = bh % a.Hk, b = bh / a.Hk;
  const int64_t one = is_k ? BwdTile<BWD_DK, NK, NV>::PARTIAL : BwdTile<BWD_DV, NK, NV>::PARTIAL;
  const float* sums = plan.partial + (is_k ? 0 : (int64_t)plan.k_blocks * plan.parts * heads * BwdTile<BWD_DK, NK, NV>::PARTIAL);
  v16f_t sum = zeros();
  if (key < w.kn) {
    for (int part = 0; part < list.parts; ++part) {
      const v4f_t* from = reinterpret_cast<const v4f_t*>(sums + (((int64_t)z * plan.parts + part) * heads + bh) * one) + (wave * width + n) * 4 * 64 + lane;
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const v4f_t x = from[g * 64];
#pragma unroll
        for (int i = 0; i < 4; ++i) sum[4 * g + i] += x[i];
      }
    }
  }
  const int64_t at = w.k_first + key + r;
  if (is_k) store_columns(reinterpret_cast<__bf16*>(a.dk) + b * a.dk_sb + hk * a.dk_sh + at * a.dk_ss, sum, a.sm_scale, n, h);
  else store_columns(reinterpret_cast<__bf16*>(a.dv) + b * a.dv_sb + hk * a.dv_sh + at * a.dv_ss, sum, 1.0f, n, h);
}

template <int NK, int NV, bool BIASED>
__global__ __launch_bounds__(256, NK > 2 ? 1 : 2) void attn_bwd_kernel(AttnBwdArgs a, AttnBwdSeqs seqs, AttnBwdPlan plan) {
  extern __shared__ __attribute__((aligned(256))) uint8_t lds[];
  const int item = (int)blockIdx.x, keys = plan.key_groups;
  if (item < keys) attn_bwd_body<BWD_DK, NK, NV, BIASED>(a, seqs, plan, item, reinterpret_cast<__bf16*>(a.dk), plan.partial, lds);
  else if (item < 2 * keys)
    attn_bwd_body<BWD_DV, NK, NV, BIASED>(a, seqs, plan, item - keys, reinterpret_cast<__bf16*>(a.dv),
                                          plan.partial + (int64_t)plan.k_blocks * plan.parts * a.B * a.Hk * BwdTile<BWD_DK, NK, NV>::PARTIAL, lds);
  else attn_bwd_body<BWD_DQ, NK, NV, BIASED>(a, seqs, plan, item - 2 * keys, reinterpret_cast<__bf16*>(a.dq), nullptr, lds);
}

template <int NK, int NV, bool BIASED>
int launch_one(const AttnBwdArgs& a, const AttnBwdSeqs& seqs, const AttnBwdPlan& plan, hipStream_t st) {
  constexpr int lds = BwdTile<BWD_DK, NK, NV>::LDS;   // the largest of the three
  static LdsLimit limit;
  if (const int rc = limit.raise((const void*)attn_bwd_kernel<NK, NV, BIASED>, lds, "attention_bwd")) return rc;
  hipLaunchKernelGGL((attn_bwd_kernel<NK, NV, BIASED>), dim3((unsigned)(2 * plan.key_groups + plan.row_groups)), dim3(256), lds, st, a, seqs, plan);
  if (const int rc = check_launch("attention_bwd")) return rc;
  if (!a.dk || plan.parts == 1) return ALTO_MXFP4_OK;
  hipLaunchKernelGGL((attn_bwd_sum_kernel<NK, NV>), dim3((unsigned)(a.B * a.Hk), (unsigned)plan.k_blocks, 2 * NK + 2 * NV), dim3(256), 0, st, a, seqs, plan);
  return check_launch("attention_bwd");
}

}  // namespace

template <int NK>
int launch_attn_bwd(const AttnBwdArgs& a, const AttnBwdSeqs& seqs, const AttnBwdPlan& plan, int64_t Dv, hipStream_t st) {
  const bool biased = a.bias || a.alibi;
  if (Dv == 64) return biased ? launch_one<NK, 1, true>(a, seqs, plan, st) : launch_one<NK, 1, false>(a, seqs, plan, st);
  return biased ? launch_one<NK, 2, true>(a, seqs, plan, st) : launch_one<NK, 2, false>(a, seqs, plan, st);
}
#endif

}  // namespace alto
