// Products of few rows of 8-bit operands with a fp32 scale for each block of 128 along the reduction (gfx950): 16 MT rows of A times 16 NT of B to a workgroup,
// whose 8 waves take every eighth block of K each and add their sums in the LDS at the end, in a fixed order.
//
// With few rows the weight is all there is to read, and what bounds a product is how much of it is under way: operands go straight from memory to the
// registers of v_mfma_f32_16x16x128_f8f6f4 (no ring, no barrier), two blocks ahead of it, in as many workgroups as 16 or 32 rows of B make.
// Measured: 1 x 14336 x 4096 13.2 us, 4.5 TB/s of the weight where a large copy has 5.2 read and written; 64 x 1024 x 4096 7.9.
// Lane (r, g) of an operand tile holds pieces of 16 bytes g and g + 4 of the block's 128 bytes of row r, of both operands alike.
#pragma once
#include "fp8.h"

namespace alto {

constexpr int FP8_ROWS_WAVES = 8;

struct Fp8RowsOperand {
  const uint8_t* codes;   // of the first row
  const float* scales;
  int64_t ld, ss_r, ss_k;
  int rows, shift;        // rows that exist from the first one on; 7: one scale for 128 rows
};

template <int MT, int NT, int CODE_A, bool B1D, typename OutT>
__device__ __forceinline__ void fp8_rows_product(const Fp8RowsOperand& A, const Fp8RowsOperand& B, int K, OutT* __restrict__ c, int64_t ldc, v4f_t* smem) {
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), r = lane & 15, g = lane >> 4;
  const int KB = (K + 127) / 128;
  auto uniform = [](const void* p) {
    const uint64_t v = reinterpret_cast<uint64_t>(p);
    return reinterpret_cast<void*>((uint64_t)__builtin_amdgcn_readfirstlane((uint32_t)(v >> 32)) << 32 | (uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)v));
  };
  const __amdgpu_buffer_rsrc_t ra = __builtin_amdgcn_make_buffer_rsrc(uniform(A.codes), 0, 0x7FFFFFFF, 0x00020000);
  const __amdgpu_buffer_rsrc_t rb = __builtin_amdgcn_make_buffer_rsrc(uniform(B.codes), 0, 0x7FFFFFFF, 0x00020000);
  // a row that does not exist: offsets out of range, zeros
  uint32_t oa[MT], ob[NT];
#pragma unroll
  for (int t = 0; t < MT; ++t) oa[t] = 16 * t + r < A.rows ? (uint32_t)(16 * t + r) * (uint32_t)A.ld + 16 * g : 0x80000000u;
#pragma unroll
  for (int u = 0; u < NT; ++u) ob[u] = 16 * u + r < B.rows ? (uint32_t)(16 * u + r) * (uint32_t)B.ld + 16 * g : 0x80000000u;
  const float *sa_at[MT], *sb_at[B1D ? 4 * NT : 1];
#pragma unroll
  for (int t = 0; t < MT; ++t) {
    const int row = 16 * t + r < A.rows ? 16 * t + r : A.rows - 1;
    sa_at[t] = A.scales + (row >> A.shift) * A.ss_r;
  }
  if constexpr (B1D) {
#pragma unroll
    for (int i = 0; i < 4 * NT; ++i) {
      const int row = 16 * (i / 4) + 4 * g + i % 4;
      sb_at[i] = B.scales + (row < B.rows ? row : B.rows - 1) * B.ss_r;
    }
  } else {
    sb_at[0] = B.scales;   // (all rows of B lie in one block of 128)
  }

  struct Block {
    v8i_t a[MT], b[NT];
    float sa[MT], sb[B1D ? 4 * NT : 1];
  };
  auto load = [&](Block& x, int k) {
    const int at = __builtin_amdgcn_readfirstlane(k * 128), rest = K - at;   // bytes of each row from there on
    const uint32_t lo = 16 * g < rest ? 0u : 0x80000000u, hi = 16 * g + 64 < rest ? 0u : 0x80000000u;
    auto operand = [&](__amdgpu_buffer_rsrc_t rsrc, uint32_t off) {
      const v4i_t p = __builtin_amdgcn_raw_buffer_load_b128(rsrc, (int)(off | lo), at, 0);
      const v4i_t q = __builtin_amdgcn_raw_buffer_load_b128(rsrc, (int)((off + 64) | hi), at, 0);
      return v8i_t{p[0], p[1], p[2], p[3], q[0], q[1], q[2], q[3]};
    };
#pragma unroll
    for (int u = 0; u < NT; ++u) x.b[u] = operand(rb, ob[u]);
#pragma unroll
    for (int t = 0; t < MT; ++t) x.a[t] = operand(ra, oa[t]);
    const int64_t ka = (int64_t)k * A.ss_k, kb = (int64_t)k * B.ss_k;
#pragma unroll
    for (int t = 0; t < MT; ++t) x.sa[t] = sa_at[t][ka];
#pragma unroll
    for (int i = 0; i < (B1D ? 4 * NT : 1); ++i) x.sb[i] = sb_at[i][kb];
  };
  v4f_t acc[MT][NT];
#pragma unroll
  for (int t = 0; t < MT; ++t)
#pragma unroll
    for (int u = 0; u < NT; ++u) acc[t][u] = v4f_t{0, 0, 0, 0};
  auto multiply = [&](Block& x, int k) {
    if ((K & 15) != 0 && k == KB - 1) {   // the last piece of a row that ends inside it: what lies behind K counts as zero
      const int rest = K - k * 128;
      auto cut = [&](v8i_t& v) {
#pragma unroll
        for (int d = 0; d < 8; ++d) {
          const int n = rest - (16 * g + 64 * (d / 4) + 4 * (d % 4));   // bytes of this dword that exist
          v[d] &= n >= 4 ? -1 : n <= 0 ? 0 : (1 << (8 * n)) - 1;
        }
      };
#pragma unroll
      for (int t = 0; t < MT; ++t) cut(x.a[t]);
#pragma unroll
      for (int u = 0; u < NT; ++u) cut(x.b[u]);
    }
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
      for (int u = 0; u < NT; ++u) {
        const v4f_t part = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(x.b[u], x.a[t], v4f_t{0, 0, 0, 0}, ALTO_FP8_E4M3, CODE_A, 0, 0, 0, 0);
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[t][u][i] = __builtin_fmaf(part[i], x.sa[t] * x.sb[B1D ? 4 * u + i : 0], acc[t][u][i]);
      }
  };
  constexpr int AHEAD = MT * NT >= (B1D ? 4 : 8) ? 2 : 4;   // blocks under way, as registers allow (64 x 4096 x 4096 with a scale for each row of both: 15.3 us with 4, which spilled, 10.9 with 2, where this
  // form of MT = 4 still keeps 11 registers in 48 bytes of scratch, eight of them read back each time round; no other form does)
  Block x[AHEAD];
  int k = wave;
#pragma unroll
  for (int j = 0; j < AHEAD; ++j)
    if (k + FP8_ROWS_WAVES * j < KB) load(x[j], k + FP8_ROWS_WAVES * j);
  for (; k < KB; k += FP8_ROWS_WAVES * AHEAD) {
#pragma unroll
    for (int j = 0; j < AHEAD; ++j) {
      const int at = k + FP8_ROWS_WAVES * j;
      if (at < KB) multiply(x[j], at);
      if (at + FP8_ROWS_WAVES * AHEAD < KB) load(x[j], at + FP8_ROWS_WAVES * AHEAD);
    }
  }
#pragma unroll
  for (int t = 0; t < MT; ++t)
#pragma unroll
    for (int u = 0; u < NT; ++u) smem[(wave * MT * NT + t * NT + u) * 64 + lane] = acc[t][u];
  __syncthreads();
  for (int i = tid; i < MT * NT * 64; i += 64 * FP8_ROWS_WAVES) {
    v4f_t sum = smem[i];
#pragma unroll
    for (int w = 1; w < FP8_ROWS_WAVES; ++w) sum += smem[w * MT * NT * 64 + i];
    const int tile = i / 64, l = i % 64, row = 16 * (tile / NT) + (l & 15), col = 16 * (tile % NT) + 4 * (l >> 4);
    if (row >= A.rows) continue;
    OutT* p = c + row * ldc + col;
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (col + e < B.rows) p[e] = (OutT)sum[e];
  }
}

}  // namespace alto
