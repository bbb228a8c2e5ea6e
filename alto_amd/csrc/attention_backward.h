// What the files of the attention backward share (attention_backward.hip: preparation and entry points; attention_backward_*.hip: the
// kernels of one head dim).
#pragma once
#include "attention.h"

namespace alto {

// Operands of the two gradient kernels.  The preparation kernel writes what comes from the workspace.
struct AttnBwdArgs {
  const uint8_t* q;             // codes [B, Hq, Sq, D/2]
  const uint8_t* k;             // codes [B, Hk, Sk, D/2]
  const uint8_t* q_scales;      // workspace: the D/32 scale bytes of every 32 rows, 8 bytes apart
  const uint8_t* k_scales;
  const __bf16* q_rows;         // workspace: the values of the codes, [B, Hq, Sq, D], [B, Hk, Sk, D], [B, Hk, Sk, Dv]
  const __bf16* k_rows;
  const __bf16* v_rows;
  const float* stats;           // workspace: of every 32 rows, 32 times lse log2(e) (+inf for a row that sees no key), then 32 times -dO . O
  const __bf16* dout;           // element (b, h, row, column) at these strides, unit stride along Dv
  int64_t do_sb, do_sh, do_ss;
  void *dq, *dk, *dv;           // bf16, the same; dq, or dk and dv, may be NULL: not wanted
  int64_t dq_sb, dq_sh, dq_ss, dk_sb, dk_sh, dk_ss, dv_sb, dv_sh, dv_ss;
  int B, Hq, Hk, Sq, Sk, Sk_used;
  float sm_scale;
  int causal;
  const float* bias;  int64_t bias_sb, bias_sh, bias_sm;
  const float* alibi; int64_t alibi_sb, alibi_sh;
};

// Sequences as AttnSeqs has them, the blocks of queries (dQ) and of keys (dK, dV) of sequence i at zq[i] and zk[i]; n = 0: B sequences of one length.
struct AttnBwdSeqs {
  int n;
  int zq[ATTN_MAX_SEQS + 1], zk[ATTN_MAX_SEQS + 1], q0[ATTN_MAX_SEQS], qn[ATTN_MAX_SEQS], k0[ATTN_MAX_SEQS], kn[ATTN_MAX_SEQS];
};

// How a launch is cut into workgroups, first those of dK and dV, then those of dQ.  A block of keys walks the tiles of 32 rows that see it, of
// all query heads on its key head; lists longer than `chunk` are dealt out to up to `parts` workgroups, whose fp32 sums meet in a kernel of
// their own (`partial`: one accumulator set for each part and block).
struct AttnBwdPlan {
  int q_blocks, k_blocks;       // over all sequences
  int parts, chunk;
  int key_groups, row_groups;   // workgroups of either kind (those of the keys: a multiple of 8)
  float* partial;
};

// Keys of one wave in the dK / dV part, rows of one in the dQ part: what 512 registers a lane hold.
constexpr int bwd_keys_sub(int) { return 1; }
constexpr int bwd_rows_sub(int) { return 1; }
inline int bwd_key_block(int64_t D) { return 128 * bwd_keys_sub((int)(D / 64)); }
inline int bwd_row_block(int64_t D) { return 128 * bwd_rows_sub((int)(D / 64)); }

template <int NK>
int launch_attn_bwd(const AttnBwdArgs& a, const AttnBwdSeqs& seqs, const AttnBwdPlan& plan, int64_t Dv, hipStream_t st);

#ifdef ALTO_ATTENTION_BACKWARD_KERNELS
namespace {

typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef short v4s_t __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) uint8_t lds_u8;
typedef __attribute__((address_space(3))) v4s_t lds_v4s;

// A tile of 32 rows of bf16 in the LDS, W columns: row after row, the 16-byte pieces of a row in an order of its own.  Two kinds of read
// take it apart: fragments along the columns (16 consecutive rows at one piece) and transposed ones (4 rows x 64 bytes); with piece c of
// row r at c ^ f(r) either kind meets all 64 banks once.  Rows of 256 bytes (or 512) need four bits of f, those of 128 (or 384) start at
// two places of the banks by themselves and need three.
template <int W>
struct RowTile {
  static constexpr int BYTES = 32 * W * 2, PR = W / 8;
  static constexpr bool WIDE = W % 128 == 0;
  static constexpr int G = WIDE ? 16 : 8;   // pieces that change places among each other
  __device__ static __forceinline__ int f(int row) { return WIDE ? (row & 3) << 2 | ((row >> 2) & 3) : (row & 2) << 1 | ((row >> 2) & 3); }
  // which byte of the 32 rows (row pitch `pitch` bytes) piece p of the tile holds
  __device__ static __forceinline__ int source(int p, int pitch) {
    const int row = p / PR, c = p % PR;
    return row * pitch + (c ^ f(row)) * 16;
  }
  // lane (r, h)'s 8 columns 16 kc + 8 h .. of row r
  __device__ static __forceinline__ int row_base(int lane) {
    const int r = lane & 31, h = lane >> 5;
    return r * (W * 2) + ((h ^ f(r)) << 4);
  }
  __device__ static __forceinline__ bf16x8_t row_frag(const uint8_t* tile, int base, int kc) {
    const int at = (base ^ ((2 * kc & (G - 1)) << 4)) + (2 * kc / G) * (G * 16);
    return *reinterpret_cast<const bf16x8_t*>(tile + at);
  }
  // lane (r, h)'s column 32 n + r of the rows 16 c + 4 h + 0..3 and 16 c + 8 + 4 h + 0..3: the order in which a score tile's registers
  // 8 c .. 8 c + 7 hold its rows.  A transposed read hands lane i of 16 the column i of four rows that the 16 lanes fetch 8 bytes each of.
  __device__ static __forceinline__ int column_base(int lane) {
    const int j = lane & 15, g = (lane >> 4) & 1, h = lane >> 5, row = 4 * h + (j >> 2);
    return row * (W * 2) + (((2 * g + ((j & 3) >> 1)) ^ f(row)) << 4) + 8 * (j & 1);
  }
  __device__ static __forceinline__ bf16x8_t column_frag(const uint8_t* tile, int base, int n, int c) {
    constexpr int N = G / 4;   // blocks of 32 columns that change places
    const int at = (base ^ ((n & (N - 1)) << 6)) + (n / N) * (N * 64) + c * (16 * W * 2);
    typedef short v8s_t __attribute__((ext_vector_type(8)));
    const v4s_t lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s*)(const __attribute__((address_space(3))) void*)(tile + at));
    const v4s_t hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s*)(const __attribute__((address_space(3))) void*)(tile + (at ^ 32) + 8 * W * 2));
    return __builtin_bit_cast(bf16x8_t, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
  }
};

// 32 rows of codes, D/2 bytes each; pieces in the order of the forward's ring
template <int NK>
struct CodeTile {
  static constexpr int D = NK * 64, BYTES = 32 * (D / 2), PR = D / 32;
  static constexpr int SW = (PR == 2 || PR == 4 || PR == 8) ? 16 / PR : 0;
  __device__ static __forceinline__ int swizzle(int row) { return SW ? (row / (SW ? SW : 1)) % PR : 0; }
  __device__ static __forceinline__ int source(int p) {
    const int row = p / PR, c = SW ? (p % PR) ^ swizzle(row) : p % PR;
    return (row * PR + c) * 16;
  }
  __device__ static __forceinline__ v8i_t frag(const uint8_t* tile, int lane, int s) {
    const int r = lane & 31, h = lane >> 5;
    return frag16(tile + r * (D / 2) + (SW ? ((32 * s + 16 * h) ^ (swizzle(r) * 16)) : 32 * s + 16 * h));
  }
};

__device__ __forceinline__ __amdgpu_buffer_rsrc_t buffer(const void* p, int64_t bytes) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(p), 0, (int)bytes, 0x00020000);
}
__device__ __forceinline__ void load_piece(__amdgpu_buffer_rsrc_t src, const uint8_t* to, int offset) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(src, (__attribute__((address_space(3))) void*)to, 16, offset, 0, 0, 0);
}

// score register v of half h <-> row 8 (v / 4) + 4 h + v % 4 of the tile
__device__ __forceinline__ int score_row(int v, int h) { return 8 * (v >> 2) + 4 * h + (v & 3); }

// eight registers of a score tile as an operand of the next product
__device__ __forceinline__ bf16x8_t pack8(const v16f_t& x, int c) {
  return __builtin_bit_cast(bf16x8_t, v4i_t{(int)pack_bf16x2(x[8 * c], x[8 * c + 1]), (int)pack_bf16x2(x[8 * c + 2], x[8 * c + 3]),
                                            (int)pack_bf16x2(x[8 * c + 4], x[8 * c + 5]), (int)pack_bf16x2(x[8 * c + 6], x[8 * c + 7])});
}

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
template <int KEYS>   // keys of a workgroup
__device__ __forceinline__ KeyList key_list(const AttnBwdArgs& a, const AttnBwdBlock& w, const AttnBwdPlan& plan) {
  KeyList l{0, 0, 0, 1};
  const int all = w.qn / 32;
  if (a.causal) {
    l.first = (w.block * KEYS - (w.kn - w.qn)) / 32;
    l.first = l.first < 0 ? 0 : l.first;
  }
  l.each = l.first < all && w.block * KEYS < w.kn ? all - l.first : 0;
  l.total = l.each * (a.Hq / a.Hk);
  l.parts = (l.total + plan.chunk - 1) / plan.chunk;
  l.parts = l.parts < 1 ? 1 : (l.parts > plan.parts ? plan.parts : l.parts);
  return l;
}

constexpr int BWD_RING = 3;

// ---------------------------------------------------------------------------------------------------------------- dK and dV
template <int NK, int NV>
struct KeysTile {
  static constexpr int CODES = CodeTile<NK>::BYTES, ROWS = RowTile<64 * NK>::BYTES, GRAD = RowTile<64 * NV>::BYTES;
  static constexpr int O_ROWS = CODES, O_GRAD = O_ROWS + ROWS, O_STATS = O_GRAD + GRAD, SLOT = O_STATS + 256;
  static constexpr int LOADS = 1 + NK + NV + (NK == 4 ? 1 : 0);   // of a wave, for one tile
  static constexpr int SUB = bwd_keys_sub(NK), KEYS = 128 * SUB;
  static constexpr int ACC = 2 * NK + 2 * NV;                                     // accumulators of 32 keys
  static constexpr int64_t PARTIAL = (int64_t)4 * SUB * ACC * 16 * 64;            // floats of a workgroup's sums
};

// Four waves own 128 SUB consecutive keys of one key head, 32 SUB each, and walk their part of the list in tiles of 32 rows.
template <int NK, int NV, bool BIASED>
__device__ __forceinline__ void attn_bwd_keys_body(const AttnBwdArgs& a, const AttnBwdSeqs& seqs, const AttnBwdPlan& plan, int item, __bf16* __restrict__ dk_out,
                                                   __bf16* __restrict__ dv_out, float* __restrict__ partial, uint8_t* ring) {
  using T = KeysTile<NK, NV>;
  using QT = RowTile<64 * NK>;
  using GT = RowTile<64 * NV>;
  constexpr int D = 64 * NK, DV = 64 * NV, SUB = T::SUB;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), r = lane & 31, h = lane >> 5;
  const int heads = a.B * a.Hk, bh = head_of(item % heads, heads);
  const int part = (item / heads) % plan.parts, z = item / heads / plan.parts;
  if (z >= plan.k_blocks) return;
  const AttnBwdBlock w = attn_bwd_block<true>(a, seqs, z);
  const KeyList list = key_list<T::KEYS>(a, w, plan);
  if (part >= list.parts) return;
  const int begin = (int)((int64_t)list.total * part / list.parts), total = (int)((int64_t)list.total * (part + 1) / list.parts) - begin;
  const int hk = bh % a.Hk, b = bh / a.Hk, group = a.Hq / a.Hk;
  const int shift = w.kn - w.qn, key0 = w.block * T::KEYS + wave * 32 * SUB;
  const int64_t k_base = (int64_t)bh * a.Sk + w.k_first;

  // the wave's keys and values stay in registers
  v8i_t kf[SUB][NK];
  int ksc[SUB][NK];
  bf16x8_t vf[SUB][4 * NV];
#pragma unroll
  for (int u = 0; u < SUB; ++u) {
    const int64_t row = k_base + (key0 + 32 * u < w.kn ? key0 + 32 * u : 0);
#pragma unroll
    for (int s = 0; s < NK; ++s) {
      kf[u][s] = frag16(a.k + (row + r) * (D / 2) + s * 32 + h * 16);
      ksc[u][s] = a.k_scales[(row / 32) * 8 + 2 * s + h];
    }
#pragma unroll
    for (int i = 0; i < 4 * NV; ++i) vf[u][i] = *reinterpret_cast<const bf16x8_t*>(a.v_rows + (row + r) * DV + 16 * i + 8 * h);
  }

  v16f_t dk[SUB][2 * NK], dv[SUB][2 * NV];
#pragma unroll
  for (int u = 0; u < SUB; ++u) {
#pragma unroll
    for (int n = 0; n < 2 * NK; ++n) dk[u][n] = zeros();
#pragma unroll
    for (int n = 0; n < 2 * NV; ++n) dv[u][n] = zeros();
  }

  const int all = w.qn / 32;
  const int own_first = a.causal ? (key0 - shift) / 32 : 0;   // the tile whose diagonal the wave's first keys are on (maybe below zero)
  const int own_whole = a.causal ? own_first + SUB : 0;       // from here on all of the wave's keys are seen
  const float c2 = a.sm_scale * ATTN_RCP_LN2;

  // each lane's part of a tile's loads
  int o_codes = 0, o_rows[NK], o_grad[NV];
  if (wave < NK) o_codes = CodeTile<NK>::source(64 * wave + lane);
#pragma unroll
  for (int j = 0; j < NK; ++j) o_rows[j] = QT::source(64 * (4 * j + wave) + lane, 2 * D);
  const int go_pitch = (int)(a.do_ss * 2);
#pragma unroll
  for (int j = 0; j < NV; ++j) o_grad[j] = GT::source(64 * (4 * j + wave) + lane, go_pitch);
  int head = 0, tile = list.first;
  if (begin > 0) { head = begin / list.each; tile += begin % list.each; }
  int next_head = head, next_tile = tile;   // of the next load
  auto fetch = [&](int slot) {
    const int hq = hk * group + next_head;
    const int64_t row = ((int64_t)b * a.Hq + hq) * a.Sq + w.q_first + 32 * next_tile;
    uint8_t* to = ring + slot * T::SLOT;
    if (wave < NK) load_piece(buffer(a.q + row * (D / 2), T::CODES), to + 1024 * wave, o_codes);
    if (NK == 4 || wave >= NK)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(buffer(a.stats + row * 2, 256), (__attribute__((address_space(3))) void*)(to + T::O_STATS), 4, lane * 4, 0, 0, 0);
    const __amdgpu_buffer_rsrc_t rows = buffer(a.q_rows + row * D, T::ROWS);
#pragma unroll
    for (int j = 0; j < NK; ++j) load_piece(rows, to + T::O_ROWS + 1024 * (4 * j + wave), o_rows[j]);
    const __amdgpu_buffer_rsrc_t grad = buffer(a.dout + b * a.do_sb + hq * a.do_sh + (int64_t)(w.q_first + 32 * next_tile) * a.do_ss, (int64_t)31 * go_pitch + 2 * DV);
#pragma unroll
    for (int j = 0; j < NV; ++j) load_piece(grad, to + T::O_GRAD + 1024 * (4 * j + wave), o_grad[j]);
    if (++next_tile == all) { next_tile = list.first; ++next_head; }
  };
  auto wait = [](bool one_in_flight) {
    if (one_in_flight) __builtin_amdgcn_s_waitcnt(0x0070 | 0x0F00 | (T::LOADS & 15));
    else __builtin_amdgcn_s_waitcnt(0x0070 | 0x0F00 | 0);
  };
  if (total > 0) fetch(0);
  if (total > 1) fetch(1);
  wait(total > 1);
  asm volatile("s_barrier" ::: "memory");

  const int row_base = GT::row_base(lane), q_col = QT::column_base(lane), g_col = GT::column_base(lane);
  int slot = 0;
  const bool live = key0 < w.kn;
  auto compute = [&](const uint8_t* at, int hq, uint32_t qs0, uint32_t qs1) {
    v16f_t S[SUB], dp[SUB];
#pragma unroll
    for (int u = 0; u < SUB; ++u) S[u] = zeros();
    static_for<NK>([&](auto sc) {
      constexpr int s = decltype(sc)::value;
      const v8i_t qf = CodeTile<NK>::frag(at, lane, s);
      const int qs = (int)((s < 2 ? qs0 : qs1) >> (8 * h));
#pragma unroll
      for (int u = 0; u < SUB; ++u) S[u] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(qf, kf[u][s], S[u], 4, 4, (2 * s) % 4, qs, 0, ksc[u][s]);
    });
    const float* stats = reinterpret_cast<const float*>(at + T::O_STATS);
    v16f_t lse2, nd;
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const v4f_t x = *reinterpret_cast<const v4f_t*>(stats + 8 * g + 4 * h), y = *reinterpret_cast<const v4f_t*>(stats + 32 + 8 * g + 4 * h);
#pragma unroll
      for (int i = 0; i < 4; ++i) { lse2[4 * g + i] = x[i]; nd[4 * g + i] = y[i]; }
    }
#pragma unroll
    for (int u = 0; u < SUB; ++u) dp[u] = nd;
#pragma unroll
    for (int kc = 0; kc < 4 * NV; ++kc) {
      const bf16x8_t gf = GT::row_frag(at + T::O_GRAD, row_base, kc);
#pragma unroll
      for (int u = 0; u < SUB; ++u) dp[u] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(gf, vf[u][kc], dp[u], 0, 0, 0);
    }
#pragma unroll
    for (int u = 0; u < SUB; ++u)
#pragma unroll
      for (int v = 0; v < 16; ++v) {
        float y = S[u][v] * c2;
        const int row = 32 * tile + score_row(v, h), key = key0 + 32 * u + r;
        if constexpr (BIASED) {
          if (a.bias) y = __builtin_fmaf(a.bias[b * a.bias_sb + hq * a.bias_sh + row * a.bias_sm + (key < w.kn ? key : 0)], ATTN_RCP_LN2, y);
          if (a.alibi) y = __builtin_fmaf(-a.alibi[b * a.alibi_sb + hq * a.alibi_sh] * ATTN_RCP_LN2, __builtin_fabsf((float)(row + shift - key)), y);
        }
        S[u][v] = y - lse2[v];
      }
    if (tile < own_whole) {
      asm volatile("" ::: "memory");   // keep this a branch: most tiles skip it
#pragma unroll
      for (int u = 0; u < SUB; ++u)
#pragma unroll
        for (int v = 0; v < 16; ++v) S[u][v] = key0 + 32 * u + r > 32 * tile + score_row(v, h) + shift ? -__builtin_inff() : S[u][v];
    }
#pragma unroll
    for (int u = 0; u < SUB; ++u)
#pragma unroll
      for (int v = 0; v < 16; ++v) S[u][v] = __builtin_amdgcn_exp2f(S[u][v]);
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      bf16x8_t p[SUB];
#pragma unroll
      for (int u = 0; u < SUB; ++u) p[u] = pack8(S[u], c);
#pragma unroll
      for (int n = 0; n < 2 * NV; ++n) {
        const bf16x8_t gf = GT::column_frag(at + T::O_GRAD, g_col, n, c);
#pragma unroll
        for (int u = 0; u < SUB; ++u) dv[u][n] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(gf, p[u], dv[u][n], 0, 0, 0);
      }
    }
#pragma unroll
    for (int u = 0; u < SUB; ++u)
#pragma unroll
      for (int v = 0; v < 16; ++v) dp[u][v] *= S[u][v];
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      bf16x8_t ds[SUB];
#pragma unroll
      for (int u = 0; u < SUB; ++u) ds[u] = pack8(dp[u], c);
#pragma unroll
      for (int n = 0; n < 2 * NK; ++n) {
        const bf16x8_t qf = QT::column_frag(at + T::O_ROWS, q_col, n, c);
#pragma unroll
        for (int u = 0; u < SUB; ++u) dk[u][n] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(qf, ds[u], dk[u][n], 0, 0, 0);
      }
    }
  };
  for (int t = 0; t < total; ++t) {
    const uint8_t* at = ring + slot * T::SLOT;
    const int hq = hk * group + head;
    const scalar_u32 qsp = scalar_ptr(a.q_scales + ((((int64_t)b * a.Hq + hq) * a.Sq + w.q_first) / 32 + tile) * 8);
    const uint32_t qs0 = qsp[0], qs1 = NK > 2 ? qsp[1] : 0;
    if (t + 2 < total) fetch(slot == 0 ? BWD_RING - 1 : slot - 1);
    if (live && tile >= own_first) compute(at, hq, qs0, qs1);
    wait(t + 2 < total);
    asm volatile("s_barrier" ::: "memory");
    slot = slot == BWD_RING - 1 ? 0 : slot + 1;
    if (++tile == all) { tile = list.first; ++head; }
  }
  if (list.parts > 1) {
    v4f_t* to = reinterpret_cast<v4f_t*>(partial + (((int64_t)z * plan.parts + part) * heads + bh) * T::PARTIAL) + wave * (SUB * T::ACC * 4 * 64) + lane;
#pragma unroll
    for (int u = 0; u < SUB; ++u)
#pragma unroll
      for (int n = 0; n < T::ACC; ++n)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const v16f_t& x = n < 2 * NK ? dk[u][n < 2 * NK ? n : 0] : dv[u][n < 2 * NK ? 0 : n - 2 * NK];
          to[((u * T::ACC + n) * 4 + g) * 64] = v4f_t{x[4 * g], x[4 * g + 1], x[4 * g + 2], x[4 * g + 3]};
        }
    return;
  }
#pragma unroll
  for (int u = 0; u < SUB; ++u) {
    const int key = key0 + 32 * u;
    if (key >= (seqs.n ? w.kn : a.Sk)) continue;
    const bool used = key < w.kn;   // keys behind the used ones get zeros
    const int64_t at = w.k_first + key + r;
#pragma unroll
    for (int n = 0; n < 2 * NK; ++n) store_columns(dk_out + b * a.dk_sb + hk * a.dk_sh + at * a.dk_ss, used ? dk[u][n] : zeros(), a.sm_scale, n, h);
#pragma unroll
    for (int n = 0; n < 2 * NV; ++n) store_columns(dv_out + b * a.dv_sb + hk * a.dv_sh + at * a.dv_ss, used ? dv[u][n] : zeros(), 1.0f, n, h);
  }
}

// Sums of the parts, in their order.  Grid: (heads, key blocks, accumulators of 32 keys); a wave has the keys that it has in the kernel above.
template <int NK, int NV>
__global__ __launch_bounds__(256) void attn_bwd_sum_kernel(AttnBwdArgs a, AttnBwdSeqs seqs, AttnBwdPlan plan) {
  using T = KeysTile<NK, NV>;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r = lane & 31, h = lane >> 5;
  const int heads = a.B * a.Hk, bh = blockIdx.x, z = blockIdx.y, n = blockIdx.z;
  const AttnBwdBlock w = attn_bwd_block<true>(a, seqs, z);
  const KeyList list = key_list<T::KEYS>(a, w, plan);
  if (list.parts == 1) return;
  const int hk = bh % a.Hk, b = bh / a.Hk;
#pragma unroll
  for (int u = 0; u < T::SUB; ++u) {
    const int key = w.block * T::KEYS + (wave * T::SUB + u) * 32;
    if (key >= (seqs.n ? w.kn : a.Sk)) continue;
    v16f_t sum = zeros();
    if (key < w.kn) {
      for (int part = 0; part < list.parts; ++part) {
        const v4f_t* from = reinterpret_cast<const v4f_t*>(plan.partial + (((int64_t)z * plan.parts + part) * heads + bh) * T::PARTIAL) + wave * (T::SUB * T::ACC * 4 * 64) +
                            (u * T::ACC + n) * 4 * 64 + lane;
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const v4f_t x = from[g * 64];
#pragma unroll
          for (int i = 0; i < 4; ++i) sum[4 * g + i] += x[i];
        }
      }
    }
    const int64_t at = w.k_first + key + r;
    if (n < 2 * NK) store_columns(reinterpret_cast<__bf16*>(a.dk) + b * a.dk_sb + hk * a.dk_sh + at * a.dk_ss, sum, a.sm_scale, n, h);
    else store_columns(reinterpret_cast<__bf16*>(a.dv) + b * a.dv_sb + hk * a.dv_sh + at * a.dv_ss, sum, 1.0f, n - 2 * NK, h);
  }
}

// ---------------------------------------------------------------------------------------------------------------------- dQ
template <int NK, int NV>
struct RowsTile {
  static constexpr int CODES = CodeTile<NK>::BYTES, ROWS = RowTile<64 * NK>::BYTES, VALUES = RowTile<64 * NV>::BYTES;
  static constexpr int O_ROWS = CODES, O_VALUES = O_ROWS + ROWS, SLOT = O_VALUES + VALUES;
  static constexpr int LOADS = 1 + NK + NV;
  static constexpr int SUB = bwd_rows_sub(NK), ROWS_WG = 128 * SUB;
};

// Four waves own 128 SUB consecutive query rows of one head, 32 SUB each, and walk the keys in tiles of 32.
template <int NK, int NV, bool BIASED>
__device__ __forceinline__ void attn_bwd_rows_body(const AttnBwdArgs& a, const AttnBwdSeqs& seqs, const AttnBwdPlan& plan, int item, __bf16* __restrict__ dq_out, uint8_t* ring) {
  using T = RowsTile<NK, NV>;
  using KT = RowTile<64 * NK>;
  using VT = RowTile<64 * NV>;
  constexpr int D = 64 * NK, DV = 64 * NV, SUB = T::SUB;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), r = lane & 31, h = lane >> 5;
  const int heads = a.B * a.Hq, bh = head_of(item % heads, heads), zi = item / heads;
  const AttnBwdBlock w = attn_bwd_block<false>(a, seqs, a.causal && !seqs.n ? plan.q_blocks - 1 - zi : zi);
  const int hq = bh % a.Hq, b = bh / a.Hq, hk = hq / (a.Hq / a.Hk);
  const int shift = w.kn - w.qn, row0 = w.block * T::ROWS_WG + wave * 32 * SUB;
  const int64_t q_base = (int64_t)bh * a.Sq + w.q_first;
  const int64_t k_base = ((int64_t)b * a.Hk + hk) * a.Sk + w.k_first;

  v8i_t qf[SUB][NK];
  int qsc[SUB][NK];
  bf16x8_t gf[SUB][4 * NV];
  float lse2[SUB], nd[SUB];
#pragma unroll
  for (int u = 0; u < SUB; ++u) {
    const int first = row0 + 32 * u < w.qn ? row0 + 32 * u : 0;
    const int64_t row = q_base + first;
#pragma unroll
    for (int s = 0; s < NK; ++s) {
      qf[u][s] = frag16(a.q + (row + r) * (D / 2) + s * 32 + h * 16);
      qsc[u][s] = a.q_scales[(row / 32) * 8 + 2 * s + h];
    }
    const __bf16* g_row = a.dout + b * a.do_sb + hq * a.do_sh + (int64_t)(w.q_first + first + r) * a.do_ss;
#pragma unroll
    for (int i = 0; i < 4 * NV; ++i) gf[u][i] = *reinterpret_cast<const bf16x8_t*>(g_row + 16 * i + 8 * h);
    lse2[u] = a.stats[row * 2 + r];
    nd[u] = a.stats[row * 2 + 32 + r];
  }

  v16f_t dq[SUB][2 * NK];
#pragma unroll
  for (int u = 0; u < SUB; ++u)
#pragma unroll
    for (int n = 0; n < 2 * NK; ++n) dq[u][n] = zeros();

  // key tiles that the wave's and the workgroup's rows see, and those that all of the wave's rows see
  const int all = w.kn / 32;
  int own = all, whole = all, total = all;
  if (a.causal) {
    whole = (row0 + shift) / 32;
    own = whole + SUB < all ? whole + SUB : all;
    const int end = (w.block + 1) * T::ROWS_WG < w.qn ? (w.block + 1) * T::ROWS_WG : w.qn;
    total = (end + shift) / 32;
  }
  if (row0 >= w.qn) own = 0;
  const float c2 = a.sm_scale * ATTN_RCP_LN2;
  const float slope2 = BIASED && a.alibi ? a.alibi[b * a.alibi_sb + hq * a.alibi_sh] * ATTN_RCP_LN2 : 0.0f;

  int o_rows[NK], o_values[NV];
  const int o_codes = CodeTile<NK>::source(64 * (wave % NK) + lane);
#pragma unroll
  for (int j = 0; j < NK; ++j) o_rows[j] = KT::source(64 * (4 * j + wave) + lane, 2 * D);
#pragma unroll
  for (int j = 0; j < NV; ++j) o_values[j] = VT::source(64 * (4 * j + wave) + lane, 2 * DV);
  auto fetch = [&](int t, int slot) {
    const int64_t row = k_base + 32 * t;
    uint8_t* to = ring + slot * T::SLOT;
    load_piece(buffer(a.k + row * (D / 2), T::CODES), to + 1024 * (wave % NK), o_codes);   // (waves past the last piece repeat one)
    const __amdgpu_buffer_rsrc_t rows = buffer(a.k_rows + row * D, T::ROWS), values = buffer(a.v_rows + row * DV, T::VALUES);
#pragma unroll
    for (int j = 0; j < NK; ++j) load_piece(rows, to + T::O_ROWS + 1024 * (4 * j + wave), o_rows[j]);
#pragma unroll
    for (int j = 0; j < NV; ++j) load_piece(values, to + T::O_VALUES + 1024 * (4 * j + wave), o_values[j]);
  };
  auto wait = [](bool one_in_flight) {
    if (one_in_flight) __builtin_amdgcn_s_waitcnt(0x0070 | 0x0F00 | (T::LOADS & 15));
    else __builtin_amdgcn_s_waitcnt(0x0070 | 0x0F00 | 0);
  };
  fetch(0, 0);
  if (total > 1) fetch(1, 1);
  wait(total > 1);
  asm volatile("s_barrier" ::: "memory");

  const int v_row = VT::row_base(lane), k_col = KT::column_base(lane);
  auto compute = [&](const uint8_t* at, int t, uint32_t ks0, uint32_t ks1) {
    v16f_t S[SUB], dp[SUB];
#pragma unroll
    for (int u = 0; u < SUB; ++u) S[u] = zeros();
    static_for<NK>([&](auto sc) {
      constexpr int s = decltype(sc)::value;
      const v8i_t kf = CodeTile<NK>::frag(at, lane, s);
      const int ks = (int)((s < 2 ? ks0 : ks1) >> (8 * h));
#pragma unroll
      for (int u = 0; u < SUB; ++u) S[u] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(kf, qf[u][s], S[u], 4, 4, (2 * s) % 4, ks, 0, qsc[u][s]);
    });
#pragma unroll
    for (int u = 0; u < SUB; ++u)
#pragma unroll
      for (int v = 0; v < 16; ++v) dp[u][v] = nd[u];
#pragma unroll
    for (int kc = 0; kc < 4 * NV; ++kc) {
      const bf16x8_t vf = VT::row_frag(at + T::O_VALUES, v_row, kc);
#pragma unroll
      for (int u = 0; u < SUB; ++u) dp[u] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(vf, gf[u][kc], dp[u], 0, 0, 0);
    }
#pragma unroll
    for (int u = 0; u < SUB; ++u)
#pragma unroll
      for (int v = 0; v < 16; ++v) {
        float y = __builtin_fmaf(S[u][v], c2, -lse2[u]);
        const int key = 32 * t + score_row(v, h), row = row0 + 32 * u + r;
        if constexpr (BIASED) {
          if (a.bias) y = __builtin_fmaf(a.bias[b * a.bias_sb + hq * a.bias_sh + (row < w.qn ? row : 0) * a.bias_sm + key], ATTN_RCP_LN2, y);
          y = __builtin_fmaf(-slope2, __builtin_fabsf((float)(row + shift - key)), y);
        }
        S[u][v] = y;
      }
    if (t >= whole) {
      asm volatile("" ::: "memory");   // keep this a branch: most tiles skip it
#pragma unroll
      for (int u = 0; u < SUB; ++u)
#pragma unroll
        for (int v = 0; v < 16; ++v) S[u][v] = 32 * t + score_row(v, h) > row0 + 32 * u + r + shift ? -__builtin_inff() : S[u][v];
    }
#pragma unroll
    for (int u = 0; u < SUB; ++u)
#pragma unroll
      for (int v = 0; v < 16; ++v) dp[u][v] *= __builtin_amdgcn_exp2f(S[u][v]);
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      bf16x8_t ds[SUB];
#pragma unroll
      for (int u = 0; u < SUB; ++u) ds[u] = pack8(dp[u], c);
#pragma unroll
      for (int n = 0; n < 2 * NK; ++n) {
        const bf16x8_t kf = KT::column_frag(at + T::O_ROWS, k_col, n, c);
#pragma unroll
        for (int u = 0; u < SUB; ++u) dq[u][n] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kf, ds[u], dq[u][n], 0, 0, 0);
      }
    }
  };
  int slot = 0;
  for (int t = 0; t < total; ++t) {
    const uint8_t* at = ring + slot * T::SLOT;
    const scalar_u32 ksp = scalar_ptr(a.k_scales + (k_base / 32 + t) * 8);
    const uint32_t ks0 = ksp[0], ks1 = NK > 2 ? ksp[1] : 0;
    if (t + 2 < total) fetch(t + 2, slot == 0 ? BWD_RING - 1 : slot - 1);
    if (t < own) compute(at, t, ks0, ks1);
    wait(t + 2 < total);
    asm volatile("s_barrier" ::: "memory");
    slot = slot == BWD_RING - 1 ? 0 : slot + 1;
  }
#pragma unroll
  for (int u = 0; u < SUB; ++u) {
    if (row0 + 32 * u >= w.qn) continue;
    __bf16* row = dq_out + b * a.dq_sb + hq * a.dq_sh + (int64_t)(w.q_first + row0 + 32 * u + r) * a.dq_ss;
#pragma unroll
    for (int n = 0; n < 2 * NK; ++n) store_columns(row, dq[u][n], a.sm_scale, n, h);
  }
}

template <int NK, int NV, bool BIASED>
__global__ __launch_bounds__(256, NK > 2 ? 1 : 2) void attn_bwd_kernel(AttnBwdArgs a, AttnBwdSeqs seqs, AttnBwdPlan plan) {
  extern __shared__ __attribute__((aligned(256))) uint8_t ring[];
  const int item = (int)blockIdx.x;
  if (item < plan.key_groups) attn_bwd_keys_body<NK, NV, BIASED>(a, seqs, plan, item, reinterpret_cast<__bf16*>(a.dk), reinterpret_cast<__bf16*>(a.dv), plan.partial, ring);
  else attn_bwd_rows_body<NK, NV, BIASED>(a, seqs, plan, item - plan.key_groups, reinterpret_cast<__bf16*>(a.dq), ring);
}

template <int NK, int NV, bool BIASED>
int launch_one(const AttnBwdArgs& a, const AttnBwdSeqs& seqs, const AttnBwdPlan& plan, hipStream_t st) {
  constexpr int slot = KeysTile<NK, NV>::SLOT > RowsTile<NK, NV>::SLOT ? KeysTile<NK, NV>::SLOT : RowsTile<NK, NV>::SLOT;
  static LdsLimit limit;
  if (const int rc = limit.raise((const void*)attn_bwd_kernel<NK, NV, BIASED>, BWD_RING * slot, "attention_bwd")) return rc;
  hipLaunchKernelGGL((attn_bwd_kernel<NK, NV, BIASED>), dim3((unsigned)(plan.key_groups + plan.row_groups)), dim3(256), BWD_RING * slot, st, a, seqs, plan);
  if (const int rc = check_launch("attention_bwd")) return rc;
  if (!a.dk || plan.parts == 1) return ALTO_MXFP4_OK;
  hipLaunchKernelGGL((attn_bwd_sum_kernel<NK, NV>), dim3((unsigned)(a.B * a.Hk), (unsigned)plan.k_blocks, KeysTile<NK, NV>::ACC), dim3(256), 0, st, a, seqs, plan);
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
