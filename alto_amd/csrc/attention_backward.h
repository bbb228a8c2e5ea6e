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

template <int NK>
int launch_attn_bwd(const AttnBwdArgs& a, const AttnBwdSeqs& seqs, int64_t Dv, int q_blocks, int k_blocks, hipStream_t st);

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
template <int N>
__device__ __forceinline__ void store_rows(__bf16* row, const v16f_t (&acc)[N], float scale, int h) {
#pragma unroll
  for (int n = 0; n < N; ++n)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const uint2 w = make_uint2(pack_bf16x2(acc[n][4 * g] * scale, acc[n][4 * g + 1] * scale), pack_bf16x2(acc[n][4 * g + 2] * scale, acc[n][4 * g + 3] * scale));
      *reinterpret_cast<uint2*>(row + 32 * n + 8 * g + 4 * h) = w;
    }
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

constexpr int BWD_RING = 3;

// ---------------------------------------------------------------------------------------------------------------- dK and dV
template <int NK, int NV>
struct KeysTile {
  static constexpr int CODES = CodeTile<NK>::BYTES, ROWS = RowTile<64 * NK>::BYTES, GRAD = RowTile<64 * NV>::BYTES;
  static constexpr int O_ROWS = CODES, O_GRAD = O_ROWS + ROWS, O_STATS = O_GRAD + GRAD, SLOT = O_STATS + 256;
  static constexpr int LOADS = 1 + NK + NV + (NK == 4 ? 1 : 0);   // of a wave, for one tile
};

// Four waves own 128 consecutive keys of one key head, 32 each, and walk the query rows of the head's group in tiles of 32.
template <int NK, int NV, bool BIASED>
__device__ __forceinline__ void attn_bwd_keys_body(const AttnBwdArgs& a, const AttnBwdSeqs& seqs, __bf16* __restrict__ dk_out, __bf16* __restrict__ dv_out, uint8_t* ring) {
  using T = KeysTile<NK, NV>;
  using QT = RowTile<64 * NK>;
  using GT = RowTile<64 * NV>;
  constexpr int D = 64 * NK, DV = 64 * NV;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), r = lane & 31, h = lane >> 5;
  const AttnBwdBlock w = attn_bwd_block<true>(a, seqs, (int)blockIdx.z);
  const int hk = blockIdx.x, b = blockIdx.y, group = a.Hq / a.Hk;
  const int shift = w.kn - w.qn, key0 = w.block * 128 + wave * 32;
  const bool live = key0 < w.kn;
  const bool stored = seqs.n ? live : key0 < a.Sk;   // keys behind the used ones get zeros
  const int64_t k_base = ((int64_t)b * a.Hk + hk) * a.Sk + w.k_first + (live ? key0 : 0);   // row of the wave's first key

  // the wave's keys and values stay in registers
  v8i_t kf[NK];
  int ksc[NK];
  bf16x8_t vf[4 * NV];
#pragma unroll
  for (int s = 0; s < NK; ++s) {
    kf[s] = frag16(a.k + (k_base + r) * (D / 2) + s * 32 + h * 16);
    ksc[s] = a.k_scales[(k_base / 32) * 8 + 2 * s + h];
  }
#pragma unroll
  for (int i = 0; i < 4 * NV; ++i) vf[i] = *reinterpret_cast<const bf16x8_t*>(a.v_rows + (k_base + r) * DV + 16 * i + 8 * h);

  v16f_t dk[2 * NK], dv[2 * NV];
#pragma unroll
  for (int n = 0; n < 2 * NK; ++n)
#pragma unroll
    for (int v = 0; v < 16; ++v) dk[n][v] = 0.0f;
#pragma unroll
  for (int n = 0; n < 2 * NV; ++n)
#pragma unroll
    for (int v = 0; v < 16; ++v) dv[n][v] = 0.0f;

  // query tiles: those that see the workgroup's first key, of every head of the group
  const int all = w.qn / 32;
  int first = 0;
  if (a.causal) {
    first = (w.block * 128 - shift) / 32;
    first = first < 0 ? 0 : first;
  }
  const int each = first < all && w.block * 128 < w.kn ? all - first : 0, total = each * group;
  const int own_first = a.causal ? (key0 - shift) / 32 : 0;   // the tile whose diagonal the wave's keys are on (maybe below zero)
  const float c2 = a.sm_scale * ATTN_RCP_LN2;

  // each lane's part of a tile's loads
  int o_codes = 0, o_rows[NK], o_grad[NV];
  if (wave < NK) o_codes = CodeTile<NK>::source(64 * wave + lane);
#pragma unroll
  for (int j = 0; j < NK; ++j) o_rows[j] = QT::source(64 * (4 * j + wave) + lane, 2 * D);
  const int go_pitch = (int)(a.do_ss * 2);
#pragma unroll
  for (int j = 0; j < NV; ++j) o_grad[j] = GT::source(64 * (4 * j + wave) + lane, go_pitch);
  int next_head = 0, next_tile = first;   // of the next load
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
    if (++next_tile == all) { next_tile = first; ++next_head; }
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
  int slot = 0, tile = first, head = 0;
  for (int t = 0; t < total; ++t) {
    const uint8_t* at = ring + slot * T::SLOT;
    const int hq = hk * group + head;
    const scalar_u32 qsp = scalar_ptr(a.q_scales + ((((int64_t)b * a.Hq + hq) * a.Sq + w.q_first) / 32 + tile) * 8);
    uint32_t qs[2] = {qsp[0], NK > 2 ? qsp[1] : 0};
    if (t + 2 < total) fetch(slot == 0 ? BWD_RING - 1 : slot - 1);
    if (live && tile >= own_first) {
      v16f_t S, P;
#pragma unroll
      for (int v = 0; v < 16; ++v) S[v] = 0.0f;
      static_for<NK>([&](auto sc) {
        constexpr int s = decltype(sc)::value;
        S = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(CodeTile<NK>::frag(at, lane, s), kf[s], S, 4, 4, (2 * s) % 4, (int)(qs[s >> 1] >> (8 * h)), 0, ksc[s]);
      });
      const float* stats = reinterpret_cast<const float*>(at + T::O_STATS);
      v16f_t dp;
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const v4f_t x = *reinterpret_cast<const v4f_t*>(stats + 32 + 8 * g + 4 * h);
#pragma unroll
        for (int i = 0; i < 4; ++i) dp[4 * g + i] = x[i];
      }
#pragma unroll
      for (int kc = 0; kc < 4 * NV; ++kc) dp = __builtin_amdgcn_mfma_f32_32x32x16_bf16(GT::row_frag(at + T::O_GRAD, row_base, kc), vf[kc], dp, 0, 0, 0);
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const v4f_t x = *reinterpret_cast<const v4f_t*>(stats + 8 * g + 4 * h);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          float y = S[4 * g + i] * c2;
          if constexpr (BIASED) {
            const int row = 32 * tile + 8 * g + 4 * h + i;
            if (a.bias) y = __builtin_fmaf(a.bias[b * a.bias_sb + hq * a.bias_sh + row * a.bias_sm + key0 + r], ATTN_RCP_LN2, y);
            if (a.alibi) y = __builtin_fmaf(-a.alibi[b * a.alibi_sb + hq * a.alibi_sh] * ATTN_RCP_LN2, __builtin_fabsf((float)(row + shift - key0 - r)), y);
          }
          S[4 * g + i] = y - x[i];
        }
      }
      if (a.causal && tile == own_first) {   // on the diagonal: key r is hidden from the rows before it
#pragma unroll
        for (int v = 0; v < 16; ++v) S[v] = score_row(v, h) < r ? -__builtin_inff() : S[v];
      }
#pragma unroll
      for (int v = 0; v < 16; ++v) P[v] = __builtin_amdgcn_exp2f(S[v]);
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const bf16x8_t p = pack8(P, c);
#pragma unroll
        for (int n = 0; n < 2 * NV; ++n) dv[n] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(GT::column_frag(at + T::O_GRAD, g_col, n, c), p, dv[n], 0, 0, 0);
      }
#pragma unroll
      for (int v = 0; v < 16; ++v) dp[v] *= P[v];
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const bf16x8_t ds = pack8(dp, c);
#pragma unroll
        for (int n = 0; n < 2 * NK; ++n) dk[n] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(QT::column_frag(at + T::O_ROWS, q_col, n, c), ds, dk[n], 0, 0, 0);
      }
    }
    wait(t + 2 < total);
    asm volatile("s_barrier" ::: "memory");
    slot = slot == BWD_RING - 1 ? 0 : slot + 1;
    if (++tile == all) { tile = first; ++head; }
  }
  if (!stored) return;
  const int64_t key = w.k_first + key0 + r;
  store_rows(dk_out + b * a.dk_sb + hk * a.dk_sh + key * a.dk_ss, dk, a.sm_scale, h);
  store_rows(dv_out + b * a.dv_sb + hk * a.dv_sh + key * a.dv_ss, dv, 1.0f, h);
}

template <int NK, int NV, bool BIASED>
__global__ __launch_bounds__(256, NK > 2 ? 1 : 2) void attn_bwd_keys_kernel(AttnBwdArgs a, AttnBwdSeqs seqs) {
  extern __shared__ __attribute__((aligned(256))) uint8_t ring[];
  attn_bwd_keys_body<NK, NV, BIASED>(a, seqs, reinterpret_cast<__bf16*>(a.dk), reinterpret_cast<__bf16*>(a.dv), ring);
}

// ---------------------------------------------------------------------------------------------------------------------- dQ
template <int NK, int NV>
struct RowsTile {
  static constexpr int CODES = CodeTile<NK>::BYTES, ROWS = RowTile<64 * NK>::BYTES, VALUES = RowTile<64 * NV>::BYTES;
  static constexpr int O_ROWS = CODES, O_VALUES = O_ROWS + ROWS, SLOT = O_VALUES + VALUES;
  static constexpr int LOADS = 1 + NK + NV;
};

// Four waves own 128 consecutive query rows of one head, 32 each, and walk the keys in tiles of 32.
template <int NK, int NV, bool BIASED>
__device__ __forceinline__ void attn_bwd_rows_body(const AttnBwdArgs& a, const AttnBwdSeqs& seqs, __bf16* __restrict__ dq_out, uint8_t* ring) {
  using T = RowsTile<NK, NV>;
  using KT = RowTile<64 * NK>;
  using VT = RowTile<64 * NV>;
  constexpr int D = 64 * NK, DV = 64 * NV;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), r = lane & 31, h = lane >> 5;
  const int z = a.causal && !seqs.n ? (int)(gridDim.z - 1 - blockIdx.z) : (int)blockIdx.z;
  const AttnBwdBlock w = attn_bwd_block<false>(a, seqs, z);
  const int hq = blockIdx.x, b = blockIdx.y, hk = hq / (a.Hq / a.Hk);
  const int shift = w.kn - w.qn, row0 = w.block * 128 + wave * 32;
  const bool live = row0 < w.qn;
  const int64_t q_base = ((int64_t)b * a.Hq + hq) * a.Sq + w.q_first + (live ? row0 : 0);
  const int64_t k_base = ((int64_t)b * a.Hk + hk) * a.Sk + w.k_first;

  v8i_t qf[NK];
  int qsc[NK];
  bf16x8_t gf[4 * NV];
#pragma unroll
  for (int s = 0; s < NK; ++s) {
    qf[s] = frag16(a.q + (q_base + r) * (D / 2) + s * 32 + h * 16);
    qsc[s] = a.q_scales[(q_base / 32) * 8 + 2 * s + h];
  }
  const __bf16* g_row = a.dout + b * a.do_sb + hq * a.do_sh + (int64_t)(w.q_first + (live ? row0 : 0) + r) * a.do_ss;
#pragma unroll
  for (int i = 0; i < 4 * NV; ++i) gf[i] = *reinterpret_cast<const bf16x8_t*>(g_row + 16 * i + 8 * h);
  const float lse2 = a.stats[q_base * 2 + r], nd = a.stats[q_base * 2 + 32 + r];

  v16f_t dq[2 * NK];
#pragma unroll
  for (int n = 0; n < 2 * NK; ++n)
#pragma unroll
    for (int v = 0; v < 16; ++v) dq[n][v] = 0.0f;

  // key tiles that the wave's and the workgroup's rows see
  const int all = w.kn / 32;
  int own = all, total = all;
  if (a.causal) {
    own = (row0 + shift) / 32 + 1;
    const int last = w.block * 128 + 96 < w.qn - 32 ? w.block * 128 + 96 : w.qn - 32;
    total = (last + shift) / 32 + 1;
  }
  if (!live) own = 0;
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
  int slot = 0;
  for (int t = 0; t < total; ++t) {
    const uint8_t* at = ring + slot * T::SLOT;
    const scalar_u32 ksp = scalar_ptr(a.k_scales + (k_base / 32 + t) * 8);
    uint32_t ks[2] = {ksp[0], NK > 2 ? ksp[1] : 0};
    if (t + 2 < total) fetch(t + 2, slot == 0 ? BWD_RING - 1 : slot - 1);
    if (t < own) {
      v16f_t S, dp;
#pragma unroll
      for (int v = 0; v < 16; ++v) S[v] = 0.0f;
      static_for<NK>([&](auto sc) {
        constexpr int s = decltype(sc)::value;
        S = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(CodeTile<NK>::frag(at, lane, s), qf[s], S, 4, 4, (2 * s) % 4, (int)(ks[s >> 1] >> (8 * h)), 0, qsc[s]);
      });
#pragma unroll
      for (int v = 0; v < 16; ++v) dp[v] = nd;
#pragma unroll
      for (int kc = 0; kc < 4 * NV; ++kc) dp = __builtin_amdgcn_mfma_f32_32x32x16_bf16(VT::row_frag(at + T::O_VALUES, v_row, kc), gf[kc], dp, 0, 0, 0);
#pragma unroll
      for (int v = 0; v < 16; ++v) {
        float y = __builtin_fmaf(S[v], c2, -lse2);
        if constexpr (BIASED) {
          const int key = 32 * t + score_row(v, h), row = row0 + r;
          if (a.bias) y = __builtin_fmaf(a.bias[b * a.bias_sb + hq * a.bias_sh + row * a.bias_sm + key], ATTN_RCP_LN2, y);
          y = __builtin_fmaf(-slope2, __builtin_fabsf((float)(row + shift - key)), y);
        }
        S[v] = y;
      }
      if (a.causal && t == own - 1) {
#pragma unroll
        for (int v = 0; v < 16; ++v) S[v] = score_row(v, h) > r ? -__builtin_inff() : S[v];
      }
#pragma unroll
      for (int v = 0; v < 16; ++v) dp[v] *= __builtin_amdgcn_exp2f(S[v]);
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const bf16x8_t ds = pack8(dp, c);
#pragma unroll
        for (int n = 0; n < 2 * NK; ++n) dq[n] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(KT::column_frag(at + T::O_ROWS, k_col, n, c), ds, dq[n], 0, 0, 0);
      }
    }
    wait(t + 2 < total);
    asm volatile("s_barrier" ::: "memory");
    slot = slot == BWD_RING - 1 ? 0 : slot + 1;
  }
  if (!live) return;
  store_rows(dq_out + b * a.dq_sb + hq * a.dq_sh + (int64_t)(w.q_first + row0 + r) * a.dq_ss, dq, a.sm_scale, h);
}

template <int NK, int NV, bool BIASED>
__global__ __launch_bounds__(256, 2) void attn_bwd_rows_kernel(AttnBwdArgs a, AttnBwdSeqs seqs) {
  extern __shared__ __attribute__((aligned(256))) uint8_t ring[];
  attn_bwd_rows_body<NK, NV, BIASED>(a, seqs, reinterpret_cast<__bf16*>(a.dq), ring);
}

template <int NK, int NV, bool BIASED>
int launch_one(const AttnBwdArgs& a, const AttnBwdSeqs& seqs, int q_blocks, int k_blocks, hipStream_t st) {
  constexpr int keys_lds = BWD_RING * KeysTile<NK, NV>::SLOT, rows_lds = BWD_RING * RowsTile<NK, NV>::SLOT;
  static LdsLimit keys_limit, rows_limit;
  if (const int rc = keys_limit.raise((const void*)attn_bwd_keys_kernel<NK, NV, BIASED>, keys_lds, "attention_bwd")) return rc;
  if (const int rc = rows_limit.raise((const void*)attn_bwd_rows_kernel<NK, NV, BIASED>, rows_lds, "attention_bwd")) return rc;
  if (a.dk) {
    hipLaunchKernelGGL((attn_bwd_keys_kernel<NK, NV, BIASED>), dim3((unsigned)a.Hk, (unsigned)a.B, (unsigned)k_blocks), dim3(256), keys_lds, st, a, seqs);
    if (const int rc = check_launch("attention_bwd")) return rc;
  }
  if (a.dq) hipLaunchKernelGGL((attn_bwd_rows_kernel<NK, NV, BIASED>), dim3((unsigned)a.Hq, (unsigned)a.B, (unsigned)q_blocks), dim3(256), rows_lds, st, a, seqs);
  return check_launch("attention_bwd");
}

}  // namespace

template <int NK>
int launch_attn_bwd(const AttnBwdArgs& a, const AttnBwdSeqs& seqs, int64_t Dv, int q_blocks, int k_blocks, hipStream_t st) {
  const bool biased = a.bias || a.alibi;
  if (Dv == 64) return biased ? launch_one<NK, 1, true>(a, seqs, q_blocks, k_blocks, st) : launch_one<NK, 1, false>(a, seqs, q_blocks, k_blocks, st);
  return biased ? launch_one<NK, 2, true>(a, seqs, q_blocks, k_blocks, st) : launch_one<NK, 2, false>(a, seqs, q_blocks, k_blocks, st);
}
#endif

}  // namespace alto
