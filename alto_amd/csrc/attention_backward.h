// What the files of the attention backward share (attention_backward.hip: preparation and entry points; attention_backward_*.hip: the
// kernels of one head dim).
#pragma once
#include "attention.h"

namespace alto {

// Operands of the gradient kernel.  "Tile": 32 rows of a head; the preparation kernel writes what comes from the workspace, tile after tile.
struct AttnBwdArgs {
  const uint8_t* q;             // codes [B, Hq, Sq, D/2]
  const uint8_t* k;             // codes [B, Hk, Sk, D/2]
  const struct QRecord* q_records;   // workspace: one of every tile
  const struct KRecord* k_records;
  const __bf16 *k_tiles, *v_tiles, *g_tiles;   // workspace: bf16 tiles (RowTile) of K and V as their codes have them, and of dO
  void *dq, *dk, *dv;           // bf16, element (b, h, row, column) at these strides, unit stride along the head dim; dq, or dk and dv, may be NULL: not wanted
  int64_t dq_sb, dq_sh, dq_ss, dk_sb, dk_sh, dk_ss, dv_sb, dv_sh, dv_ss;
  int B, Hq, Hk, Sq, Sk, Sk_used;
  float sm_scale;
  int causal;
  const float* bias;  int64_t bias_sb, bias_sh, bias_sm;   // bias_sm below 2^24
  int distances;                // the records' slopes count
};

// Where 16-byte piece `p` of row `row` (columns 8 p .. 8 p + 7) sits in a tile of bf16 rows: the 32 rows' pieces of the same columns side by side,
// the rows in groups of four that change places from piece to piece.  Two kinds of read take a tile apart: fragments along the columns (16
// consecutive rows at one piece) and transposed ones (4 rows x 64 bytes); either meets all banks of the LDS once, and all of a tile's
// fragments sit at constant distances from one or two addresses a lane.
__host__ __device__ __forceinline__ constexpr int tile_piece(int row, int p) { return p * 32 + (row ^ ((p & 3) << 2)); }

// What a tile has besides its rows.  The scale byte of columns 64 s + 32 h .. + 32 is at 4 h + s, the order of the score products.
struct KRecord {
  uint8_t scales[8], unused[8];
};
struct QRecord {
  float lse2[32], minus_d[32];   // lse log2(e) (+inf for a row that sees no key), -dO . O
  uint8_t scales[8];
  float slope;                   // -slope / sm_scale of the head
  float unused;
};

// Sequences as AttnSeqs has them, the blocks of queries (dQ) and of keys (dK, dV) of sequence i at zq[i] and zk[i]; n = 0: B sequences of one length.
struct AttnBwdSeqs {
  int n;
  int zq[ATTN_MAX_SEQS + 1], zk[ATTN_MAX_SEQS + 1], q0[ATTN_MAX_SEQS], qn[ATTN_MAX_SEQS], k0[ATTN_MAX_SEQS], kn[ATTN_MAX_SEQS];
};

// How a launch is cut into workgroups, those of dK and dV and those of dQ, the longer ones first.  A block of keys walks the tiles of 32 rows that see it, of
// all query heads on its key head, a block of rows the tiles of 32 keys that it sees; lists longer than `chunk` are dealt out to up to `parts`
// workgroups, whose fp32 sums meet in a kernel of their own (`partial`: one set of accumulators for each part and block).
struct AttnBwdCut {
  int parts, chunk;
  float* partial;
};
struct AttnBwdPlan {
  int q_blocks, k_blocks;       // over all sequences
  AttnBwdCut keys, rows;
  int key_groups, row_groups;   // workgroups of either kind (multiples of 8: the last few may have nothing)
  int rows_first;
  int key_sums, row_sums;       // workgroups of the kernel that adds the parts
};
// Waves of a workgroup, each with 32 keys or query rows; two workgroups share a compute unit where 256 registers a lane do.  (One of 8 waves reads each
// tile half as often, but its two waves on a SIMD keep step and wait together: 4 x 2048 tokens, 64 / 8 heads of 128, 988 us for 889.)
constexpr int BWD_WAVES = 4, BWD_BLOCK = 32 * BWD_WAVES;

template <int NK>
int launch_attn_bwd(const AttnBwdArgs& a, const AttnBwdSeqs& seqs, const AttnBwdPlan& plan, int64_t Dv, hipStream_t st);

__device__ __forceinline__ float e8m0_value(uint32_t e) { return u2f(e ? e << 23 : 0x00400000u); }

// eight codes of one dword as bf16
__device__ __forceinline__ v4i_t decode8(uint32_t codes, float scale) {
  return v4i_t{__builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 0)), __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 1)),
               __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 2)), __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 3))};
}

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

__device__ __forceinline__ void load_dword(__amdgpu_buffer_rsrc_t src, const uint8_t* to, int lane_offset, int offset) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(src, (__attribute__((address_space(3))) void*)to, 4, lane_offset, offset, 0, 0);
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

// All of these in accumulation registers at one time (nothing is emitted).  Above head dims of 128, where a lane has 512 registers, half of them for
// accumulators, the compiler otherwise gives the scores the place of sums that it moves out and back in every step: up to 128 of 530 instructions, 378
// us for 343 (2048 tokens, 64 / 8 heads of 192 / 128).
#define ALTO_A2(x, i) "+a"(x[i]), "+a"(x[i + 1])
template <int NK>
__device__ __forceinline__ void at_once(v16f_t& s, v16f_t (&k)[NK]) {
  if constexpr (NK == 6) asm volatile("" : "+a"(s), ALTO_A2(k, 0), ALTO_A2(k, 2), ALTO_A2(k, 4));
  if constexpr (NK == 8) asm volatile("" : "+a"(s), ALTO_A2(k, 0), ALTO_A2(k, 2), ALTO_A2(k, 4), ALTO_A2(k, 6));
}
template <int NV, int NK>
__device__ __forceinline__ void at_once(v16f_t& s, v16f_t (&v)[NV], v16f_t (&k)[NK]) {
  if constexpr (NV == 2 && NK == 6) asm volatile("" : "+a"(s), ALTO_A2(v, 0), ALTO_A2(k, 0), ALTO_A2(k, 2), ALTO_A2(k, 4));
  if constexpr (NV == 4 && NK == 6) asm volatile("" : "+a"(s), ALTO_A2(v, 0), ALTO_A2(v, 2), ALTO_A2(k, 0), ALTO_A2(k, 2), ALTO_A2(k, 4));
  if constexpr (NV == 2 && NK == 8) asm volatile("" : "+a"(s), ALTO_A2(v, 0), ALTO_A2(k, 0), ALTO_A2(k, 2), ALTO_A2(k, 4), ALTO_A2(k, 6));
  if constexpr (NV == 4 && NK == 8) asm volatile("" : "+a"(s), ALTO_A2(v, 0), ALTO_A2(v, 2), ALTO_A2(k, 0), ALTO_A2(k, 2), ALTO_A2(k, 4), ALTO_A2(k, 6));
}
#undef ALTO_A2

// A wave's 32 rows of W columns of transposed accumulators as bf16 to memory, by way of `lds` (64 W bytes of the wave's own, idle): written straight from
// the registers they would be 16 bytes a row and store, and a store passes one line of the cache at a time.  The 16-byte pieces of a row change
// places with the row, so that the writes of 32 rows meet all banks.
template <int W>
__device__ __forceinline__ void store_rows(const v16f_t* acc, float scale, bool live, uint8_t* lds, __bf16* to, int64_t stride, int lane) {
  const int r = lane & 31, h = lane >> 5;
#pragma unroll
  for (int n = 0; n < W / 32; ++n)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const uint2 w = make_uint2(pack_bf16x2(acc[n][4 * g] * scale, acc[n][4 * g + 1] * scale), pack_bf16x2(acc[n][4 * g + 2] * scale, acc[n][4 * g + 3] * scale));
      *reinterpret_cast<uint2*>(lds + r * 2 * W + ((4 * n + g) ^ (r & 7)) * 16 + 8 * h) = live ? w : make_uint2(0, 0);
    }
  wave_lds_order();
#pragma unroll
  for (int k = 0; k < W / 16; ++k) {
    const int i = 64 * k + lane, row = i / (W / 8), piece = i % (W / 8);
    *reinterpret_cast<v4i_t*>(to + row * stride + 8 * piece) = *reinterpret_cast<const v4i_t*>(lds + row * 2 * W + (piece ^ (row & 7)) * 16);
  }
  wave_lds_order();
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

// Workgroup `item` of heads x each: its (batch, head) pair and its place among that pair's, the longest of all pairs first.  Eight neighbouring
// workgroups go to the eight XCDs in turn: each XCD gets a range of consecutive pairs, so that a head's operands come into one L2.  (One pair after the
// other in each XCD misses less in the L2 while it lasts, but ends with the last pair's longest: 4 x 2048 tokens, 64 / 8 heads of 128, 943 us for 889.)
struct HeadItem {
  int head, index;
};
__device__ __forceinline__ HeadItem head_item(int item, int heads) {
  const int o = item % heads;
  return {heads % 8 == 0 ? (o & 7) * (heads >> 3) + (o >> 3) : o, item / heads};
}

// Part `part` of a list of `total` tiles: tiles begin .. + count of it, of `parts` in all (none behind these).
struct BwdPart {
  int begin, count, parts;
};
__device__ __forceinline__ BwdPart part_of(int total, int part, const AttnBwdCut& cut) {
  int parts = (total + cut.chunk - 1) / cut.chunk;
  parts = parts < 1 ? 1 : (parts > cut.parts ? cut.parts : parts);
  const int begin = (int)((int64_t)total * part / parts);
  return {begin, (int)((int64_t)total * (part + 1) / parts) - begin, parts};
}
// The list of a block of keys: tiles first .. + each of every head of the group.
struct KeyList {
  int first, each, total;
};
__device__ __forceinline__ KeyList key_list(const AttnBwdArgs& a, const AttnBwdBlock& w) {
  KeyList l{0, 0, 0};
  const int all = w.qn / 32;
  if (a.causal) {
    l.first = (w.block * BWD_BLOCK - (w.kn - w.qn)) / 32;
    l.first = l.first < 0 ? 0 : l.first;
  }
  l.each = l.first < all && w.block * BWD_BLOCK < w.kn ? all - l.first : 0;
  l.total = l.each * (a.Hq / a.Hk);
  return l;
}
// Block `z` of rows in the order of dispatch (the longest lists first), and the length of its list.
__device__ __forceinline__ AttnBwdBlock row_block(const AttnBwdArgs& a, const AttnBwdSeqs& seqs, const AttnBwdPlan& plan, int z) {
  return attn_bwd_block<false>(a, seqs, a.causal && !seqs.n ? plan.q_blocks - 1 - z : z);
}
__device__ __forceinline__ int row_list(const AttnBwdArgs& a, const AttnBwdBlock& w) {
  if (!a.causal) return w.kn / 32;
  const int end = (w.block + 1) * BWD_BLOCK < w.qn ? (w.block + 1) * BWD_BLOCK : w.qn;
  return (end + w.kn - w.qn) / 32;
}

// What the two kinds of workgroup share (dK and dV in one of them: as two kinds, each with scores of its own, they took more).  A wave holds 32 rows of its own side (keys for dK and dV, query rows for dQ) and walks tiles of 32 rows of
// the other side, from which it takes
//   the codes, for the scores        S = codes x own codes                  (rows of the tile in registers, its own in lanes),
//   bf16 rows, for dP                dO x own V, or V x own dO,
//   bf16 rows by columns, as the factor of its sums   dV += P^T dO and dK += dS^T Q, or dQ += dS K.
// A tile comes into the LDS by loads without registers in between, 1 KB each, dealt out to the waves.
template <int NK, int NV>
struct BwdShape {
  static constexpr int CODES = CodeTile<NK>::BYTES, ROWS_D = RowTile<64 * NK>::BYTES, ROWS_V = RowTile<64 * NV>::BYTES;
  static constexpr int ACC = 2 * NK + 2 * NV;                                 // accumulators of 32 keys
  // Sums of part `part` of block z of head `bh`: of every wave its accumulators, four registers of all lanes after the other
  template <int N>
  __device__ static __forceinline__ v4f_t* sums(const AttnBwdCut& cut, int z, int part, int heads, int bh, int wave, int lane) {
    return reinterpret_cast<v4f_t*>(cut.partial) + ((((int64_t)z * cut.parts + part) * heads + bh) * BWD_WAVES + wave) * (N * 4 * 64) + lane;
  }
};

struct BwdPlace {
  int tile, at;   // a tile's number in its sequence, and among all of its side
};

// A tile's codes and its record (in a slot of 1 KB), one load of 64 pieces of 16 bytes a wave; with D = 256 two.  Waves behind the codes' pieces all take
// the record: where a wave loads from and to is settled before the loop, and no step has a branch for it.
template <bool KEYS, int NK>
struct BwdSmall {
  static constexpr int LOADS = NK == 4 ? 2 : 1, CODES = CodeTile<NK>::BYTES, RECORD = KEYS ? sizeof(QRecord) : sizeof(KRecord);
  const uint8_t *codes, *records, *from;
  int bytes, offset;      // of what this wave loads first: a tile's, and this lane's in it
  bool takes_codes;
  int to, slot_bytes, second_to;   // slots of this wave's in the LDS
  __device__ __forceinline__ BwdSmall(const uint8_t* codes, const void* all_records, int wave, int lane, int lds_codes, int lds_records)
      : codes(codes), records(reinterpret_cast<const uint8_t*>(all_records)) {
    takes_codes = wave < NK;
    from = takes_codes ? codes : records;
    bytes = takes_codes ? CODES : RECORD;
    offset = takes_codes ? CodeTile<NK>::source(64 * wave + lane) : 16 * lane;
    to = takes_codes ? lds_codes + 1024 * wave : lds_records;
    slot_bytes = takes_codes ? CODES : 1024;
    second_to = lds_records;
  }
  // of `n` tiles from `first` on
  __device__ __forceinline__ __amdgpu_buffer_rsrc_t source(int64_t first, int n) const { return buffer(from + first * bytes, (int64_t)n * bytes); }
  __device__ __forceinline__ __amdgpu_buffer_rsrc_t second(int64_t first, int n) const { return buffer(records + first * RECORD, (int64_t)n * RECORD); }
  // tile `t` of these, to these slots
  __device__ __forceinline__ void operator()(__amdgpu_buffer_rsrc_t source, __amdgpu_buffer_rsrc_t second, int t, const uint8_t* lds, int code_slot, int record_slot, int lane) const {
    load_piece(source, lds + to + (takes_codes ? code_slot : record_slot) * slot_bytes, offset, (int)((uint32_t)t * bytes));
    if constexpr (LOADS == 2) load_piece(second, lds + second_to + record_slot * 1024, 16 * lane, (int)((uint32_t)t * RECORD));
  }
};
// Load `l` of tile `t` of bf16 rows (as many of each wave as it is wide / 64)
template <int W>
__device__ __forceinline__ void load_rows(__amdgpu_buffer_rsrc_t source, const uint8_t* to, int t, int l, int wave, int lane) {
  load_piece(source, to + 1024 * (BWD_WAVES * l + wave), lane * 16 + 1024 * wave, (int)((uint32_t)t * RowTile<W>::BYTES + 1024 * BWD_WAVES * l));
}
template <int W>
__device__ __forceinline__ __amdgpu_buffer_rsrc_t rows_source(const __bf16* tiles, int64_t first, int n) {
  return buffer(reinterpret_cast<const uint8_t*>(tiles) + first * RowTile<W>::BYTES, (int64_t)n * RowTile<W>::BYTES);
}
template <int N>   // loads that may stay under way
__device__ __forceinline__ void wait_all_but() { __builtin_amdgcn_s_waitcnt(0x0070 | 0x0F00 | (N & 15) | (N >> 4) << 14); }
template <int N>   // ... but no read or write of the LDS
__device__ __forceinline__ void wait_lds_and_all_but() { __builtin_amdgcn_s_waitcnt(0x0070 | (N & 15) | (N >> 4) << 14); }

// What is added to the scores: nothing; slopes times distances; a bias, and distances (of slope 0 where there are none).  A score tile's additive terms,
// over sm_scale, are what its accumulators start with: the rest of a step does not know of them.
enum { ADD_NOTHING, ADD_DISTANCES, ADD_BIAS };

// A wave's 32 x 32 block of the bias in the LDS, 4 KB of its own: one dword a lane and load straight from memory, which asks nothing of the bias'
// alignment and needs no register on the way.  (Read element by element where it is used, the same bias made the whole backward of 3 x 8 heads, 480
// rows, 1056 keys of 192 / 128 three times as long: 181 us for 61 without it.)  Register 4 g + e of lane (r, h) takes the element 8 g + 4 h + e of
// the side that is in the registers and r of the other.
template <bool KEYS>
struct BiasBlock {
  static constexpr int LOADS = 16, BYTES = 4096;
  // in: the block's first element
  __device__ static __forceinline__ void load(const float* in, int64_t row_stride, const uint8_t* to, int lane) {
    const int stride = 4 * (int)row_stride;
    const __amdgpu_buffer_rsrc_t src = buffer(in, 0x7FFFFFFF);
#pragma unroll
    for (int l = 0; l < LOADS; ++l) {
      if constexpr (KEYS) {   // 4 rows x 16 keys, in the order of the reading lanes
        load_dword(src, to + 256 * l, (lane & 3) * stride + (lane >> 2) * 4, (4 * (l >> 1)) * stride + 64 * (l & 1));
      } else {                // 2 rows x 32 keys, pieces of four keys in an order that changes with the row
        load_dword(src, to + 256 * l, (lane >> 5) * stride + ((4 * (lane & 31)) ^ ((l & 7) << 4)), 2 * l * stride);
      }
    }
  }
  __device__ static __forceinline__ v4f_t read(const uint8_t* at, int lane, int g) {
    if constexpr (KEYS) return *reinterpret_cast<const v4f_t*>(at + 1024 * g + 16 * lane);
    const int r = lane & 31, h = lane >> 5;
    return *reinterpret_cast<const v4f_t*>(at + 128 * r + 16 * ((2 * g + h) ^ ((r >> 1) & 7)));
  }
};

// A probability.  None is above 1; where the bias is so large that lse has no bits left for the scores, a rounding could say so.  NaN stays NaN
// (v_minimum3_f32: 72 us for 3 x 8 heads, 480 rows, 1056 keys of 192 / 128; the clamp that v_exp_f32 has for nothing, 70 us, makes 0 of it, and dV would
// not see a NaN of the bias or of lse).
template <int ADD>
__device__ __forceinline__ float probability_of(float x, std::integral_constant<int, ADD>) {
  const float p = __builtin_amdgcn_exp2f(x);
  return ADD == ADD_BIAS ? __builtin_elementwise_minimum(p, 1.0f) : p;
}

// The products of a step are issued in a fixed order (sched_barrier): the read of an operand runs AHEAD products before its use, vector work lies
// behind each product.  Left to itself the compiler puts every read right in front of its product and waits there.  Four products where the registers
// allow it (2 x 1024 tokens, 16 heads of 64 with slopes 41.1 us, two 42.4; 8192 tokens, 16 / 2 heads of 256 / 128 1246, 1261), two with D = 128.
constexpr int bwd_ahead(int nk) { return nk == 2 ? 2 : 4; }

// ---------------------------------------------------------------------------------------------------------------- dK and dV
// Four slots of codes, statistics and scales, three of dO, two of Q's values, which the workgroup makes from the codes one step ahead (a quarter of the
// bytes to fetch).
template <int NK, int NV>
struct KeysLds {
  using T = BwdShape<NK, NV>;
  static constexpr int O_V = 4 * T::CODES, O_D = O_V + 3 * T::ROWS_V, O_RECORD = O_D + 2 * T::ROWS_D, O_BIAS = O_RECORD + 4 * 1024;
};
// One step: S and dP of a tile, its probabilities, and its part of the sums.  P is taken from S behind the products of dP, dS behind those of dV.
template <int NK, int NV, int ADD>
__device__ __forceinline__ void attn_bwd_keys_body(const AttnBwdArgs& a, const AttnBwdSeqs& seqs, const AttnBwdPlan& plan, int item, __bf16* __restrict__ dk_out,
                                                   __bf16* __restrict__ dv_out, uint8_t* lds) {
  using T = BwdShape<NK, NV>;
  using VT = RowTile<64 * NV>;
  using DT = RowTile<64 * NK>;
  using L = KeysLds<NK, NV>;
  using Small = BwdSmall<true, NK>;
  using Bias = BiasBlock<true>;
  constexpr int D = 64 * NK;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), r = lane & 31, h = lane >> 5;
  const int heads = a.B * a.Hk, group = a.Hq / a.Hk;
  const HeadItem it = head_item(item, heads);
  const int bh = it.head, part = it.index % plan.keys.parts, z = it.index / plan.keys.parts;
  if (z >= plan.k_blocks) return;   // (the last few of a number that is no multiple of 8)
  const AttnBwdBlock w = attn_bwd_block<true>(a, seqs, z);
  const KeyList list = key_list(a, w);
  const BwdPart mine = part_of(list.total, part, plan.keys);
  if (part >= mine.parts) return;
  const int begin = mine.begin, total = mine.count;
  const int b = bh / a.Hk, hk = bh % a.Hk;
  const int shift = w.kn - w.qn, key0 = w.block * BWD_BLOCK + wave * 32;
  const bool live = key0 < w.kn;
  const int own_tile = bh * (a.Sk / 32) + w.k_first / 32 + (live ? key0 / 32 : 0);

  v16f_t dk[2 * NK], dv[2 * NV];
#pragma unroll
  for (int n = 0; n < 2 * NK; ++n) dk[n] = zeros();
#pragma unroll
  for (int n = 0; n < 2 * NV; ++n) dv[n] = zeros();

  if (total > 0) {
    v8i_t xf[NK];
    bf16x8_t yf[4 * NV];
#pragma unroll
    for (int s = 0; s < NK; ++s) xf[s] = frag16(a.k + ((int64_t)own_tile * 32 + r) * (D / 2) + s * 32 + h * 16);
    const uint32_t x_scales = *reinterpret_cast<const uint32_t*>(a.k_records[own_tile].scales + 4 * h);
    const uint8_t* y = reinterpret_cast<const uint8_t*>(a.v_tiles) + (int64_t)own_tile * T::ROWS_V;
#pragma unroll
    for (int i = 0; i < 4 * NV; ++i) yf[i] = VT::row_frag(y + VT::row_base(lane, i & 1), i);

    const int tiles = a.Sq / 32, last = w.qn / 32;
    int next_tile = list.first, left = total, next_base = (b * a.Hq + hk * group) * tiles + w.q_first / 32;
    if (begin > 0) {
      next_base += begin / list.each * tiles;
      next_tile += begin % list.each;
    }
    auto next = [&]() {   // (past the end: the last tile again)
      const BwdPlace p{next_tile, next_base + next_tile};
      const int more = left - 1 < 1 ? left - 1 : 1;
      left -= more;
      next_tile += more;
      const int wrap = next_tile == last ? -1 : 0;
      next_tile += wrap & (list.first - last);
      next_base += wrap & tiles;
      return p;
    };
    const Small small(a.q, a.q_records, wave, lane, 0, L::O_RECORD);
    auto record = [&](int i) { return reinterpret_cast<const QRecord*>(lds + L::O_RECORD + (i & 3) * 1024); };
    const int code_base = lane * 16, row_base[2] = {VT::row_base(lane, 0), VT::row_base(lane, 1)}, column_base[2] = {VT::column_base(lane, 0), VT::column_base(lane, 1)};
    const float c2 = a.sm_scale * ATTN_RCP_LN2, inverse_scale = 1.0f / a.sm_scale;
    // The additive terms of tile `i`
    v16f_t S;
    uint8_t* const at_bias = lds + L::O_BIAS + wave * Bias::BYTES;
    auto load_bias = [&](const BwdPlace& p) {
      const int hq = p.at / tiles - b * a.Hq;
      Bias::load(a.bias + b * a.bias_sb + hq * a.bias_sh + (int64_t)(32 * p.tile) * a.bias_sm + (live ? key0 : 0), a.bias_sm, at_bias, lane);
    };
    auto read_bias = [&](int g) {
      const v4f_t x = Bias::read(at_bias, lane, g);
#pragma unroll
      for (int e = 0; e < 4; ++e) S[4 * g + e] = x[e];
    };
    auto add = [&](const BwdPlace& p, int i, int g) {
      const float slope = record(i)->slope, away = (float)(32 * p.tile + 4 * h + shift - key0 - r);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float x = slope * __builtin_fabsf(away + (float)(8 * g + e));
        S[4 * g + e] = ADD == ADD_BIAS ? __builtin_fmaf(S[4 * g + e], inverse_scale, x) : x;
      }
    };
    // Eight columns of one row of tile `i`'s values, from its codes: dword j = 2 wave + h + 8 u of row r
    uint32_t eight = 0, eight_scales = 0;
    const int eight_from = 16 * r + 4 * h, eight_to = tile_piece(r, 2 * wave + h) * 16;
    auto read_codes = [&](int i, int u) {
      eight = *reinterpret_cast<const uint32_t*>(lds + (i & 3) * T::CODES + ((wave >> 1) + 2 * u) * 512 + 8 * (wave & 1) + eight_from);
      eight_scales = reinterpret_cast<const uint32_t*>(record(i)->scales)[wave >> 1];
    };
    auto write_values = [&](int i, int u) {
      *reinterpret_cast<v4i_t*>(lds + L::O_D + (i & 1) * T::ROWS_D + 4096 * u + eight_to) = decode8(eight, e8m0_value((eight_scales >> (8 * u)) & 0xFFu));
    };
    auto load_small = [&](const BwdPlace& p, int i) { small(small.source(p.at, 1), small.second(p.at, 1), 0, lds, i & 3, i & 3, lane); };
    auto load_grads = [&](const BwdPlace& p, int l, int slot) { load_rows<64 * NV>(rows_source<64 * NV>(a.g_tiles, p.at, 1), lds + L::O_V + slot * T::ROWS_V, 0, l, wave, lane); };

    BwdPlace p0 = next(), p1 = next(), p2 = next();
    if constexpr (ADD == ADD_BIAS) load_bias(p0);
    load_small(p0, 0);
    load_small(p1, 1);
#pragma unroll
    for (int l = 0; l < NV; ++l) load_grads(p0, l, 0);
#pragma unroll
    for (int l = 0; l < NV; ++l) load_grads(p1, l, 1);
    load_small(p2, 2);
    wait_all_but<NV + Small::LOADS>();
    asm volatile("s_barrier" ::: "memory");
#pragma unroll
    for (int u = 0; u < NK; ++u) {
      read_codes(0, u);
      write_values(0, u);
    }
    if constexpr (ADD != ADD_NOTHING) {
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        if constexpr (ADD == ADD_BIAS) read_bias(g);
        add(p0, 0, g);
      }
    }
    __builtin_amdgcn_s_waitcnt(0xC07F);   // lgkmcnt(0)
    asm volatile("s_barrier" ::: "memory");
    if constexpr (ADD == ADD_BIAS) load_bias(p1);

    constexpr int NS = NK, NI = 4 * NV, NF = 4 * NV, NG = 4 * NK, N = NS + NI + NF + NG, AHEAD = bwd_ahead(NK);
    int slot = 0;
    for (int t = 0; t < total; ++t) {
      const int two_on = slot == 0 ? 2 : slot - 1;
      const BwdPlace p3 = next();
      const uint8_t* const at_codes = lds + (t & 3) * T::CODES + code_base;
      const uint8_t *at_rows[2], *at_v[2], *at_d[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        at_rows[i] = lds + L::O_V + slot * T::ROWS_V + row_base[i];
        at_v[i] = lds + L::O_V + slot * T::ROWS_V + column_base[i];
        at_d[i] = lds + L::O_D + (t & 1) * T::ROWS_D + column_base[i];
      }
      const QRecord* const rec = record(t);
      if constexpr (ADD == ADD_NOTHING) S = zeros();
      v16f_t dp;
      v4f_t l4[2];
      bf16x8_t frag[AHEAD + 1];
      uint32_t pk[8], dsk[8];
      auto read = [&](auto ic) {
        constexpr int i = decltype(ic)::value;
        if constexpr (i < N) {
          bf16x8_t& x = frag[i % (AHEAD + 1)];
          if constexpr (i < NS) x = *reinterpret_cast<const bf16x8_t*>(at_codes + i * 1024);
          else if constexpr (i < NS + NI) x = VT::row_frag(at_rows[(i - NS) & 1], i - NS);
          else if constexpr (i < NS + NI + NF) x = VT::column_frag(at_v[0], at_v[1], (i - NS - NI) % (2 * NV), (i - NS - NI) / (2 * NV));
          else x = DT::column_frag(at_d[0], at_d[1], (i - NS - NI - NF) % (2 * NK), (i - NS - NI - NF) / (2 * NK));
        }
      };
      auto four = [](const uint32_t (&o)[8], int c) { return __builtin_bit_cast(bf16x8_t, v4i_t{(int)o[4 * c], (int)o[4 * c + 1], (int)o[4 * c + 2], (int)o[4 * c + 3]}); };
      const uint32_t sc = reinterpret_cast<const uint32_t*>(rec->scales)[h];
      auto product = [&](auto ic) {
        constexpr int i = decltype(ic)::value;
        const bf16x8_t& x = frag[i % (AHEAD + 1)];
        if constexpr (i < NS) {
          const v4i_t q = __builtin_bit_cast(v4i_t, x);
          S = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(v8i_t{q[0], q[1], q[2], q[3], 0, 0, 0, 0}, xf[i], S, 4, 4, i, (int)sc, i, (int)x_scales);
        } else if constexpr (i < NS + NI) {
          dp = __builtin_amdgcn_mfma_f32_32x32x16_bf16(x, yf[i - NS], dp, 0, 0, 0);
        } else if constexpr (i < NS + NI + NF) {
          constexpr int j = i - NS - NI, n = j % (2 * NV), c = j / (2 * NV);
          dv[n] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(x, four(pk, c), dv[n], 0, 0, 0);
        } else {
          constexpr int j = i - NS - NI - NF, n = j % (2 * NK), c = j / (2 * NK);
          dk[n] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(x, four(dsk, c), dk[n], 0, 0, 0);
        }
      };
      auto read_stats = [&](int g) { l4[g & 1] = *reinterpret_cast<const v4f_t*>(rec->lse2 + 8 * g + 4 * h); };
      auto probability = [&](int i) {   // of the pair of rows i
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const int v = 2 * i + k;
          S[v] = probability_of(__builtin_fmaf(S[v], c2, -l4[(v >> 2) & 1][v & 3]), std::integral_constant<int, ADD>{});
        }
        if ((i & 1) == 1 && i / 2 + 2 < 4) read_stats(i / 2 + 2);   // (the group's last use is behind us)
      };
      auto pack_p = [&](int i) { pk[i] = pack_bf16x2(S[2 * i], S[2 * i + 1]); };
      auto pack_ds = [&](int i) { dsk[i] = pack_bf16x2(S[2 * i] * dp[2 * i], S[2 * i + 1] * dp[2 * i + 1]); };
      __builtin_amdgcn_sched_barrier(0);
      static_for<AHEAD>([&](auto ic) { read(ic); });
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const v4f_t x = *reinterpret_cast<const v4f_t*>(rec->minus_d + 8 * g + 4 * h);
#pragma unroll
        for (int i = 0; i < 4; ++i) dp[4 * g + i] = x[i];
      }
      read_stats(0);
      read_stats(1);
      __builtin_amdgcn_sched_barrier(0);
      static_for<N>([&](auto ic) {
        constexpr int i = decltype(ic)::value;
        read(std::integral_constant<int, i + AHEAD>{});
        if constexpr (ADD == ADD_BIAS && i == NS + NI + NF) wait_all_but<0>();   // the last step's loads, the bias of the next tile among them
        product(ic);
        if constexpr (i == NS - 1) {
          if constexpr (NK > 2) {
            at_once(S, dv, dk);
            asm volatile("" : "+v"(S));
          }
          if (a.causal && 32 * p0.tile + shift <= key0) {   // the diagonal's tile, or one before it, that another wave of the workgroup needs
            asm volatile("" ::: "memory");   // keep this a branch: most tiles skip it
            const int hidden = key0 + r - 32 * p0.tile - shift;
#pragma unroll
            for (int v = 0; v < 16; ++v) S[v] = score_row(v, h) < hidden ? -__builtin_inff() : S[v];
          }
        }
        // vector work
        if constexpr (i >= NS && i < NS + NI) {
          constexpr int j = i - NS, u0 = 8 * j / NI, u1 = 8 * (j + 1) / NI;
#pragma unroll
          for (int u = u0; u < u1; ++u) probability(u);
#pragma unroll
          for (int u = u0; u < u1; ++u)
            if (u > 0) pack_p(u - 1);
          if constexpr (j == NI - 1) pack_p(7);
        }
        if constexpr (i >= NS + NI && i < NS + NI + NF) {
          constexpr int j = i - NS - NI, first = NF / 4, u0 = j < first ? 0 : 8 * (j - first) / (NF - first), u1 = j < first ? 0 : 8 * (j - first + 1) / (NF - first);
#pragma unroll
          for (int u = u0; u < u1; ++u) pack_ds(u);
        }
        if constexpr (i >= NS + NI + NF) {   // the loads for later tiles, the next one's values
          constexpr int j = i - NS - NI - NF;
          if constexpr (j == 0) load_small(p3, t + 3);
          if constexpr (j >= 1 && j <= NV) load_grads(p2, j - 1, two_on);
          if constexpr (j % 4 == 0) read_codes(t + 1, j / 4);
          if constexpr (j % 4 == 3) write_values(t + 1, j / 4);
          if constexpr (ADD == ADD_BIAS && j < 2) {
            read_bias(2 * j);
            read_bias(2 * j + 1);
          }
          if constexpr (ADD != ADD_NOTHING && (j == 2 || j == 3)) {
            add(p1, t + 1, 2 * (j - 2));
            add(p1, t + 1, 2 * (j - 2) + 1);
            if constexpr (ADD == ADD_BIAS && j == 3) load_bias(p2);   // (where the block lay that has just been read)
          }
        }
        __builtin_amdgcn_sched_barrier(0);
      });
      p0 = p1;
      p1 = p2;
      p2 = p3;
      slot = slot == 2 ? 0 : slot + 1;
      wait_lds_and_all_but<Small::LOADS + NV + (ADD == ADD_BIAS ? Bias::LOADS : 0)>();   // all but this step's loads; the values are written
      asm volatile("s_barrier" ::: "memory");
    }
    wait_lds_and_all_but<0>();   // (the last loads into the LDS, which nobody reads, before it is used otherwise)
  }

  if (mine.parts > 1) {
    v4f_t* to = T::template sums<T::ACC>(plan.keys, z, part, heads, bh, wave, lane);
#pragma unroll
    for (int n = 0; n < T::ACC; ++n)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const v16f_t& x = n < 2 * NK ? dk[n < 2 * NK ? n : 0] : dv[n < 2 * NK ? 0 : n - 2 * NK];
        to[(n * 4 + g) * 64] = v4f_t{x[4 * g], x[4 * g + 1], x[4 * g + 2], x[4 * g + 3]};
      }
    return;
  }
  asm volatile("s_barrier" ::: "memory");   // (no wave's loads or reads are under way any more)
  if (key0 >= (seqs.n ? w.kn : a.Sk)) return;
  const int64_t at = w.k_first + key0;   // (keys behind the used ones: zeros)
  uint8_t* const own = lds + wave * (64 * 64 * (NK > NV ? NK : NV));
  store_rows<64 * NK>(dk, a.sm_scale, live, own, dk_out + b * a.dk_sb + hk * a.dk_sh + at * a.dk_ss, a.dk_ss, lane);
  store_rows<64 * NV>(dv, 1.0f, live, own, dv_out + b * a.dv_sb + hk * a.dv_sh + at * a.dv_ss, a.dv_ss, lane);
}

// Sums of the parts, in their order.  A workgroup: 32 columns of one block's gradients (dK, then dV; those of dQ behind them).
template <int NK, int NV>
__global__ __launch_bounds__(64 * BWD_WAVES) void attn_bwd_sum_kernel(AttnBwdArgs a, AttnBwdSeqs seqs, AttnBwdPlan plan) {
  using T = BwdShape<NK, NV>;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r = lane & 31, h = lane >> 5;
  auto sum_of = [&](auto count, const AttnBwdCut& cut, int parts, int z, int heads, int bh, int n) {
    v16f_t sum = zeros();
#pragma unroll 4
    for (int part = 0; part < parts; ++part) {   // (the loads of four parts at a time under way)
      const v4f_t* from = T::template sums<decltype(count)::value>(cut, z, part, heads, bh, wave, lane) + n * 4 * 64;
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const v4f_t x = from[g * 64];
#pragma unroll
        for (int i = 0; i < 4; ++i) sum[4 * g + i] += x[i];
      }
    }
    return sum;
  };
  int item = blockIdx.x;
  if (item < plan.key_sums) {
    const int heads = a.B * a.Hk, n = item % T::ACC, bh = item / T::ACC % heads, z = item / T::ACC / heads;
    const AttnBwdBlock w = attn_bwd_block<true>(a, seqs, z);
    const int parts = part_of(key_list(a, w).total, 0, plan.keys).parts, key = w.block * BWD_BLOCK + wave * 32;
    if (parts == 1 || key >= (seqs.n ? w.kn : a.Sk)) return;
    const v16f_t sum = sum_of(std::integral_constant<int, T::ACC>{}, plan.keys, key < w.kn ? parts : 0, z, heads, bh, n);
    const int hk = bh % a.Hk, b = bh / a.Hk;
    const int64_t at = w.k_first + key + r;
    if (n < 2 * NK) store_columns(reinterpret_cast<__bf16*>(a.dk) + b * a.dk_sb + hk * a.dk_sh + at * a.dk_ss, sum, a.sm_scale, n, h);
    else store_columns(reinterpret_cast<__bf16*>(a.dv) + b * a.dv_sb + hk * a.dv_sh + at * a.dv_ss, sum, 1.0f, n - 2 * NK, h);
    return;
  }
  item -= plan.key_sums;
  const int heads = a.B * a.Hq, n = item % (2 * NK), bh = item / (2 * NK) % heads, z = item / (2 * NK) / heads;
  const AttnBwdBlock w = row_block(a, seqs, plan, z);
  const int parts = part_of(row_list(a, w), 0, plan.rows).parts, row = w.block * BWD_BLOCK + wave * 32;
  if (parts == 1 || row >= w.qn) return;
  const v16f_t sum = sum_of(std::integral_constant<int, 2 * NK>{}, plan.rows, parts, z, heads, bh, n);
  store_columns(reinterpret_cast<__bf16*>(a.dq) + (bh / a.Hq) * a.dq_sb + (bh % a.Hq) * a.dq_sh + (int64_t)(w.q_first + row + r) * a.dq_ss, sum, a.sm_scale, n, h);
}

// ---------------------------------------------------------------------------------------------------------------------- dQ
template <int NK, int NV>
struct RowsLds {   // three slots of codes, V and K, four of scales
  using T = BwdShape<NK, NV>;
  static constexpr int O_V = 3 * T::CODES, O_D = O_V + 3 * T::ROWS_V, O_RECORD = O_D + 3 * T::ROWS_D, O_BIAS = O_RECORD + 4 * 1024;
};
// Three stages in one step: S and dP of tile t + 1 and the sums' product with tile t - 1 on the matrix pipe, dS of tile t on the vector pipe.
template <int NK, int NV, int ADD>
__device__ __forceinline__ void attn_bwd_rows_body(const AttnBwdArgs& a, const AttnBwdSeqs& seqs, const AttnBwdPlan& plan, int item, __bf16* __restrict__ dq_out, uint8_t* lds) {
  using T = BwdShape<NK, NV>;
  using VT = RowTile<64 * NV>;
  using DT = RowTile<64 * NK>;
  constexpr int D = 64 * NK;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), r = lane & 31, h = lane >> 5;
  using L = RowsLds<NK, NV>;
  using Small = BwdSmall<false, NK>;
  using Bias = BiasBlock<false>;
  const int heads = a.B * a.Hq;
  const HeadItem it = head_item(item, heads);
  const int bh = it.head, b = bh / a.Hq, hq = bh % a.Hq, hk = hq / (a.Hq / a.Hk);
  const int part = it.index % plan.rows.parts, z = it.index / plan.rows.parts;
  if (z >= plan.q_blocks) return;
  const AttnBwdBlock w = row_block(a, seqs, plan, z);
  const BwdPart mine = part_of(row_list(a, w), part, plan.rows);
  if (part >= mine.parts) return;
  const int shift = w.kn - w.qn, row0 = w.block * BWD_BLOCK + wave * 32, begin = mine.begin, total = mine.count;   // tile t of this part: begin + t
  const bool live = row0 < w.qn;
  const int own_tile = bh * (a.Sq / 32) + w.q_first / 32 + (live ? row0 / 32 : 0), first_at = (b * a.Hk + hk) * (a.Sk / 32) + w.k_first / 32 + begin;

  v16f_t acc[2 * NK];
#pragma unroll
  for (int n = 0; n < 2 * NK; ++n) acc[n] = zeros();
  v8i_t xf[NK];
  bf16x8_t yf[4 * NV];
  v16f_t nd;
#pragma unroll
  for (int s = 0; s < NK; ++s) xf[s] = frag16(a.q + ((int64_t)own_tile * 32 + r) * (D / 2) + s * 32 + h * 16);
  const QRecord* const own_record = a.q_records + own_tile;
  const uint32_t x_scales = *reinterpret_cast<const uint32_t*>(own_record->scales + 4 * h);
  const uint8_t* y0 = reinterpret_cast<const uint8_t*>(a.g_tiles) + (int64_t)own_tile * T::ROWS_V;
#pragma unroll
  for (int i = 0; i < 4 * NV; ++i) yf[i] = VT::row_frag(y0 + VT::row_base(lane, i & 1), i);
  const float lse2 = own_record->lse2[r], minus_d = own_record->minus_d[r];
#pragma unroll
  for (int v = 0; v < 16; ++v) nd[v] = minus_d;
  const float c2 = a.sm_scale * ATTN_RCP_LN2, inverse_scale = 1.0f / a.sm_scale;
  const float slope = ADD == ADD_NOTHING ? 0.0f : own_record->slope;

  const Small small(a.k, a.k_records, wave, lane, 0, L::O_RECORD);
  const int code_base = lane * 16, row_base[2] = {VT::row_base(lane, 0), VT::row_base(lane, 1)}, column_base[2] = {DT::column_base(lane, 0), DT::column_base(lane, 1)};
  auto tile = [&](int t) { return t < total ? t : total - 1; };   // (past the end: the last tile again)
  // (a head's rows take less than 4 GB)
  const __amdgpu_buffer_rsrc_t small_source = small.source(first_at, total), second_source = small.second(first_at, total);
  const __amdgpu_buffer_rsrc_t v_source = rows_source<64 * NV>(a.v_tiles, first_at, total), k_source = rows_source<64 * NK>(a.k_tiles, first_at, total);

  // Which keys of the tile the lane's row sees, in the bits of the packed pairs: most tiles are seen whole (state 2), the diagonal's in part (1), a
  // tile behind it not at all (0: another wave of the workgroup needs it).
  uint32_t seen[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) seen[i] = ~0u;
  int state = 2;
  auto look = [&](int tile) {
    if (!a.causal) return;
    const int away = row0 + shift - 32 * (begin + tile);   // a multiple of 32
    const int now = away > 0 ? 2 : (away == 0 ? 1 : 0);
    if (now == state) return;
    state = now;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int x = score_row(2 * i, h);   // the pair's first key; the second is the next one
      seen[i] = now == 2 ? ~0u : (now == 1 ? (x <= r ? 0xFFFFu : 0u) | (x + 1 <= r ? 0xFFFF0000u : 0u) : 0u);
    }
  };

  // The products in order: those of the scores, then by turns one of dP and one of the sums.
  constexpr int NS = NK, NI = 4 * NV, NF = 4 * NK, AHEAD = bwd_ahead(NK), HALVES = 16, STEP_LOADS = Small::LOADS + NV + NK;
  struct Op {
    int kind, j;   // 0: S, 1: dP, 2: sums
  };
  struct Scores {
    v16f_t S, dp;
  };
  // The additive terms of tile `i`, in the registers where its scores will be
  uint8_t* const at_bias = lds + L::O_BIAS + wave * Bias::BYTES;
  auto load_bias = [&](int i) {
    Bias::load(a.bias + b * a.bias_sb + hq * a.bias_sh + (int64_t)(live ? row0 : 0) * a.bias_sm + 32 * (begin + tile(i)), a.bias_sm, at_bias, lane);
  };
  auto add = [&](int i, int g, v16f_t& S) {
    const float away = (float)(row0 + r + shift - 32 * (begin + i) - 4 * h);
    v4f_t x;
    if constexpr (ADD == ADD_BIAS) x = Bias::read(at_bias, lane, g);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float y = slope * __builtin_fabsf(away - (float)(8 * g + e));
      S[4 * g + e] = ADD == ADD_BIAS ? __builtin_fmaf(x[e], inverse_scale, y) : y;
    }
  };
  // (RUN: the first step only has scores to compute)
  auto step = [&](auto run, int t, int slot, Scores& from, const bf16x8_t (&f)[2], Scores& to, bf16x8_t (&f_next)[2]) {
    constexpr bool RUN = decltype(run)::value;
    const int after = slot == 2 ? 0 : slot + 1, before = slot == 0 ? 2 : slot - 1;
    const uint8_t* const at_codes = lds + after * T::CODES + code_base;
    const uint8_t *at_rows[2], *at_columns[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      at_rows[i] = lds + L::O_V + after * T::ROWS_V + row_base[i];
      at_columns[i] = lds + L::O_D + before * T::ROWS_D + column_base[i];
    }
    constexpr int N = RUN ? NS + NI + NF : NS + NI;
    auto op = [](int i) constexpr {
      if (i < NS) return Op{0, i};
      if (!RUN) return Op{1, i - NS};
      int inner = 0, factor = 0;
      for (int k = NS;; ++k) {
        const bool take_inner = inner < NI && (factor == NF || inner * NF <= factor * NI);
        if (k == i) return take_inner ? Op{1, inner} : Op{2, factor};
        if (take_inner) ++inner; else ++factor;
      }
    };
    const uint32_t sc = reinterpret_cast<const uint32_t*>(lds + L::O_RECORD + ((t + 1) & 3) * 1024)[h];
    bf16x8_t frag[AHEAD + 1];
    auto read = [&](auto ic) {
      constexpr int i = decltype(ic)::value;
      if constexpr (i < N) {
        constexpr Op o = op(i);
        bf16x8_t& x = frag[i % (AHEAD + 1)];
        if constexpr (o.kind == 0) x = *reinterpret_cast<const bf16x8_t*>(at_codes + o.j * 1024);
        else if constexpr (o.kind == 1) x = VT::row_frag(at_rows[o.j & 1], o.j);
        else x = DT::column_frag(at_columns[0], at_columns[1], o.j % (2 * NK), o.j / (2 * NK));
      }
    };
    auto product = [&](auto ic) {
      constexpr int i = decltype(ic)::value;
      constexpr Op o = op(i);
      const bf16x8_t& x = frag[i % (AHEAD + 1)];
      if constexpr (o.kind == 0) {
        const v4i_t q = __builtin_bit_cast(v4i_t, x);
        to.S = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(v8i_t{q[0], q[1], q[2], q[3], 0, 0, 0, 0}, xf[o.j], ADD == ADD_NOTHING && o.j == 0 ? zeros() : to.S, 4, 4, o.j, (int)sc, o.j, (int)x_scales);
      } else if constexpr (o.kind == 1) {
        to.dp = __builtin_amdgcn_mfma_f32_32x32x16_bf16(x, yf[o.j], o.j == 0 ? nd : to.dp, 0, 0, 0);
      } else {
        acc[o.j % (2 * NK)] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(x, f[o.j / (2 * NK)], acc[o.j % (2 * NK)], 0, 0, 0);
      }
    };
    // dS of tile t, a pair of keys at a time, in two halves
    float e[8][2];
    uint32_t out[8];
    auto half = [&](auto uc) {
      constexpr int u = decltype(uc)::value, i = u >> 1;
      if constexpr ((u & 1) == 0) {
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const int v = 2 * i + k;
          e[i][k] = probability_of(__builtin_fmaf(from.S[v], c2, -lse2), std::integral_constant<int, ADD>{});
        }
      } else {
        out[i] = pack_bf16x2(e[i][0] * from.dp[2 * i], e[i][1] * from.dp[2 * i + 1]) & seen[i];
        asm volatile("" : "+v"(out[i]));   // (here: otherwise it is moved behind the step, to where it is used)
        if constexpr (ADD != ADD_NOTHING && (i & 1) == 1) {
          if constexpr (ADD == ADD_BIAS && i == 1) wait_all_but<STEP_LOADS>();   // the last step's loads, the bias of tile t + 2 among them
          add(t + 2, i >> 1, from.S);
        }
      }
    };
    __builtin_amdgcn_sched_barrier(0);
    static_for<AHEAD>([&](auto ic) { read(ic); });
    __builtin_amdgcn_sched_barrier(0);
    static_for<N>([&](auto ic) {
      constexpr int i = decltype(ic)::value;
      read(std::integral_constant<int, i + AHEAD>{});
      product(ic);
      if constexpr (NK > 2 && RUN && i == NS - 1) at_once(to.S, acc);
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

  // Loads go out two steps before they are used: a step starts those of the scores of t + 3 and the factor of t + 1, and ends with a wait for
  // everything that earlier steps started.
  auto load_scores = [&](int i, int slot) {
    const int t = tile(i);
    small(small_source, second_source, t, lds, slot, i & 3, lane);
#pragma unroll
    for (int l = 0; l < NV; ++l) load_rows<64 * NV>(v_source, lds + L::O_V + slot * T::ROWS_V, t, l, wave, lane);
  };
  auto load_factor = [&](int i, int slot) {
    const int t = tile(i);
#pragma unroll
    for (int l = 0; l < NK; ++l) load_rows<64 * NK>(k_source, lds + L::O_D + slot * T::ROWS_D, t, l, wave, lane);
  };
  Scores x, y;
  if constexpr (ADD == ADD_BIAS) {
    load_bias(0);
    wait_all_but<0>();
  }
  if constexpr (ADD != ADD_NOTHING) {
#pragma unroll
    for (int g = 0; g < 4; ++g) add(0, g, x.S);
  }
  if constexpr (ADD == ADD_BIAS) {
    __builtin_amdgcn_s_waitcnt(0xC07F);   // lgkmcnt(0): the block is read
    load_bias(1);
    wait_all_but<0>();
  }
  if constexpr (ADD != ADD_NOTHING) {
#pragma unroll
    for (int g = 0; g < 4; ++g) add(1, g, y.S);
  }
  if constexpr (ADD == ADD_BIAS) {
    __builtin_amdgcn_s_waitcnt(0xC07F);
    load_bias(2);
  }
  load_scores(0, 0);
  load_factor(0, 0);
  load_factor(0, 2);   // (what the first step multiplies with zeros)
  load_scores(1, 1);
  load_scores(2, 2);
  wait_all_but<Small::LOADS + NV>();
  asm volatile("s_barrier" ::: "memory");
  bf16x8_t f[2], g[2];
  f[0] = f[1] = __builtin_bit_cast(bf16x8_t, v4i_t{0, 0, 0, 0});
  step(std::false_type{}, -1, 2, x, f, x, f);
  asm volatile("s_barrier" ::: "memory");   // (every wave has read tile 0, whose slot the next step's loads go to)
  int slot = 0;   // of tile t
  auto whole_step = [&](int t, Scores& from, const bf16x8_t (&f_now)[2], Scores& to, bf16x8_t (&f_next)[2]) {
    const int after = slot == 2 ? 0 : slot + 1;
    load_scores(t + 3, slot);
    load_factor(t + 1, after);
    look(t);
    step(std::true_type{}, t, slot, from, f_now, to, f_next);
    slot = after;
    if constexpr (ADD == ADD_BIAS) {
      __builtin_amdgcn_s_waitcnt(0xC07F);
      load_bias(t + 3);   // (where the block lay that has just been read)
    }
    wait_all_but<STEP_LOADS + (ADD == ADD_BIAS ? Bias::LOADS : 0)>();
    asm volatile("s_barrier" ::: "memory");
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
  {   // the last tile's sums
    const uint8_t* at = lds + L::O_D + (slot == 0 ? 2 : slot - 1) * T::ROWS_D;
#pragma unroll
    for (int c = 0; c < 2; ++c)
#pragma unroll
      for (int n = 0; n < 2 * NK; ++n) acc[n] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(DT::column_frag(at + column_base[0], at + column_base[1], n, c), f[c], acc[n], 0, 0, 0);
  }
  wait_lds_and_all_but<0>();   // (this wave's reads; the last loads into the LDS, which nobody reads, before it is used otherwise)
  if (mine.parts > 1) {
    if (!live) return;
    v4f_t* to = T::template sums<2 * NK>(plan.rows, z, part, heads, bh, wave, lane);
#pragma unroll
    for (int n = 0; n < 2 * NK; ++n)
#pragma unroll
      for (int g = 0; g < 4; ++g) to[(n * 4 + g) * 64] = v4f_t{acc[n][4 * g], acc[n][4 * g + 1], acc[n][4 * g + 2], acc[n][4 * g + 3]};
    return;
  }
  asm volatile("s_barrier" ::: "memory");   // (no wave's loads or reads are under way any more)
  if (!live) return;
  store_rows<64 * NK>(acc, a.sm_scale, true, lds + wave * (64 * 64 * NK), dq_out + b * a.dq_sb + hq * a.dq_sh + (int64_t)(w.q_first + row0) * a.dq_ss, a.dq_ss, lane);
}

// All three gradients in one launch, so that the workgroups of dQ fill the units while the last ones of dK and dV end.
//
// 4 x 2048 tokens of 128, 64 / 8 heads, causal: 730 to 800 us for 687 GFLOP (five products over the pairs that the mask leaves), 0.9 PFLOP/s; it issues 44
// products of 32 cycles for every 32 x 32 scores of either side (26 for dK and dV, 18 for dQ, four of them on codes), matrix pipes busy 61 % of the cycles,
// vector pipes 45 %, some instruction issued in 89 %, at a clock of 1.7 GHz that is 2.1 when fewer products are busy: the clock and the waits bound it
// together, which of them more has not been told apart.  K's, V's and Q's tiles are read as codes or once for four waves, nothing is spilled.  With D = 64 the
// issue of instructions is the bound (99 % of the cycles), with D > 128 one wave a SIMD waits for itself (54 %).
template <int NK, int NV, int ADD>
__global__ __launch_bounds__(64 * BWD_WAVES, NK > 2 ? 1 : 2) void attn_bwd_kernel(AttnBwdArgs a, AttnBwdSeqs seqs, AttnBwdPlan plan) {
  extern __shared__ __attribute__((aligned(256))) uint8_t lds[];
  const int at = (int)blockIdx.x;
  const bool rows = plan.rows_first ? at < plan.row_groups : at >= plan.key_groups;
  const int item = rows == (plan.rows_first != 0) ? at : at - (rows ? plan.key_groups : plan.row_groups);
  if (!rows) attn_bwd_keys_body<NK, NV, ADD>(a, seqs, plan, item, reinterpret_cast<__bf16*>(a.dk), reinterpret_cast<__bf16*>(a.dv), lds);
  else attn_bwd_rows_body<NK, NV, ADD>(a, seqs, plan, item, reinterpret_cast<__bf16*>(a.dq), lds);
}

template <int NK, int NV, int ADD>
int launch_one(const AttnBwdArgs& a, const AttnBwdSeqs& seqs, const AttnBwdPlan& plan, hipStream_t st) {
  using T = BwdShape<NK, NV>;
  constexpr int keys = KeysLds<NK, NV>::O_BIAS, rows = RowsLds<NK, NV>::O_BIAS, lds = (keys > rows ? keys : rows) + (ADD == ADD_BIAS ? BWD_WAVES * 4096 : 0);
  static LdsLimit limit;
  if (const int rc = limit.raise((const void*)attn_bwd_kernel<NK, NV, ADD>, lds, "attention_bwd")) return rc;
  hipLaunchKernelGGL((attn_bwd_kernel<NK, NV, ADD>), dim3((unsigned)(plan.key_groups + plan.row_groups)), dim3(64 * BWD_WAVES), lds, st, a, seqs, plan);
  if (const int rc = check_launch("attention_bwd")) return rc;
  AttnBwdPlan sums = plan;
  sums.key_sums *= T::ACC;
  sums.row_sums *= 2 * NK;
  if (sums.key_sums + sums.row_sums == 0) return ALTO_MXFP4_OK;
  hipLaunchKernelGGL((attn_bwd_sum_kernel<NK, NV>), dim3((unsigned)(sums.key_sums + sums.row_sums)), dim3(64 * BWD_WAVES), 0, st, a, seqs, sums);
  return check_launch("attention_bwd");
}

}  // namespace

template <int NK>
int launch_attn_bwd(const AttnBwdArgs& a, const AttnBwdSeqs& seqs, const AttnBwdPlan& plan, int64_t Dv, hipStream_t st) {
  const int add = a.bias ? ADD_BIAS : (a.distances ? ADD_DISTANCES : ADD_NOTHING);
  auto one = [&](auto nv) {
    constexpr int NV = decltype(nv)::value;
    switch (add) {
      case ADD_BIAS: return launch_one<NK, NV, ADD_BIAS>(a, seqs, plan, st);
      case ADD_DISTANCES: return launch_one<NK, NV, ADD_DISTANCES>(a, seqs, plan, st);
      default: return launch_one<NK, NV, ADD_NOTHING>(a, seqs, plan, st);
    }
  };
  return Dv == 64 ? one(std::integral_constant<int, 1>{}) : one(std::integral_constant<int, 2>{});
}
#endif

}  // namespace alto
