// Rotation of Q and K by their tokens' positions (gfx950), both in one launch.
//
// Of every head's D columns the first R are rotated in pairs, (x_i, x_{i + R/2}) or interleaved (x_{2i}, x_{2i+1}), i < R/2, by the angle
// a = position * inv_freq_i:   y1 = c x1 - s x2,  y2 = s x1 + c x2,  c = factor cos a,  s = factor sin a;   the others pass.  The rotation's
// transpose (s -> -s) is its backward.
//
// What bounds it is HBM: Q and K read and written once.  Angles belong to a token, not to a head: a workgroup takes up to ROTARY_TOKENS tokens (some of the heads
// of one, where there are few tokens), computes their R/2 cosines and sines once, in 64 bits (a position of a million times a frequency has
// lost its fraction in 32), and keeps them as fp32 in the LDS while it streams the heads.  No table: nothing to keep, to size or to read, and
// any position is as good as any other.  4 x 2048 tokens of 64 + 8 heads of 128 in bf16 take 63 us either way, 4.8 TB/s (a copy of as many bytes: 5.1);
// 16 tokens of 32 + 8 heads 3.8 us, most of it the launch and one round to memory.
#include "common.h"

namespace alto {
namespace {

constexpr int ROTARY_TOKENS = 8;   // most of a workgroup

struct RotaryOperand {
  const void* x;
  void* y;
  int64_t x_sb, x_sh, x_ss, y_sb, y_sh, y_ss;   // element strides of batch, head, row; unit stride along D
};
struct RotaryArgs {
  RotaryOperand q, k;
  const double* inv_freq;
  const void* positions;        // element (b, s) at b pos_sb + s pos_ss; NULL: s
  int64_t pos_sb, pos_ss;
  int pos_is_32;
  double cos_factor, sin_factor;
  int64_t tokens;               // B S
  int S, Hq, Hk, D, R;
  int per_group, heads_each;    // tokens of a workgroup; heads of one (of Q's, then K's)
};

// cos and sin of a in 64 bits: a minus the nearest multiple of pi/2 (pi/2 in two parts), then their Taylor polynomials on [-pi/4, pi/4] (the
// first terms left out are below 2e-13 there).
__device__ __forceinline__ void cos_sin(double a, double& c, double& s) {
  const double n = __builtin_rint(a * 0.63661977236758134308);
  double r = __builtin_fma(-n, 1.57079632679489655800, a);
  r = __builtin_fma(-n, 6.12323399573676603587e-17, r);
  const double z = r * r;
  double ps = -1.0 / 1307674368000.0;
  ps = __builtin_fma(ps, z, 1.0 / 6227020800.0);
  ps = __builtin_fma(ps, z, -1.0 / 39916800.0);
  ps = __builtin_fma(ps, z, 1.0 / 362880.0);
  ps = __builtin_fma(ps, z, -1.0 / 5040.0);
  ps = __builtin_fma(ps, z, 1.0 / 120.0);
  ps = __builtin_fma(ps, z, -1.0 / 6.0);
  const double sn = __builtin_fma(ps * z, r, r);
  double pc = 1.0 / 20922789888000.0;
  pc = __builtin_fma(pc, z, -1.0 / 87178291200.0);
  pc = __builtin_fma(pc, z, 1.0 / 479001600.0);
  pc = __builtin_fma(pc, z, -1.0 / 3628800.0);
  pc = __builtin_fma(pc, z, 1.0 / 40320.0);
  pc = __builtin_fma(pc, z, -1.0 / 720.0);
  pc = __builtin_fma(pc, z, 1.0 / 24.0);
  const double cn = __builtin_fma(z * z, pc, __builtin_fma(z, -0.5, 1.0));
  const int quarter = (int)((int64_t)n & 3);
  const double u = quarter & 1 ? sn : cn, v = quarter & 1 ? cn : sn;
  c = quarter == 1 || quarter == 2 ? -u : u;
  s = quarter >= 2 ? -v : v;
}

// VEC consecutive elements
template <typename T, int VEC>
struct Vec {
  T x[VEC] __attribute__((aligned(sizeof(T) * VEC)));
};
template <typename T, int VEC>
__device__ __forceinline__ void load(const T* p, float (&f)[VEC]) {
  const Vec<T, VEC> v = *reinterpret_cast<const Vec<T, VEC>*>(p);
#pragma unroll
  for (int i = 0; i < VEC; ++i) f[i] = (float)v.x[i];
}
template <typename T, int VEC>
__device__ __forceinline__ void store(T* p, const float (&f)[VEC]) {
  Vec<T, VEC> v;
#pragma unroll
  for (int i = 0; i < VEC; ++i) v.x[i] = (T)f[i];
  *reinterpret_cast<Vec<T, VEC>*>(p) = v;
}

// Unit `u` of a head's work: VEC pairs (half: VEC columns of either half; interleaved: 2 VEC neighbouring columns), or behind the `turned` ones 2 VEC
// columns that pass (the last may be VEC of them).  table: the token's R/2 cosines, then its sines.
template <typename T, int VEC, bool INTERLEAVED>
__device__ __forceinline__ void rotate_unit(const T* x, T* y, const float* table, int half, int R, int D, int u, int turned) {
  if (u >= turned) {
    const int c = R + (u - turned) * 2 * VEC;
    *reinterpret_cast<Vec<T, VEC>*>(y + c) = *reinterpret_cast<const Vec<T, VEC>*>(x + c);
    if (c + VEC < D) *reinterpret_cast<Vec<T, VEC>*>(y + c + VEC) = *reinterpret_cast<const Vec<T, VEC>*>(x + c + VEC);
    return;
  }
  const float* cs = table + u * VEC;
  const int c1 = INTERLEAVED ? 2 * u * VEC : u * VEC, c2 = INTERLEAVED ? c1 + VEC : c1 + half;
  float p[VEC], q[VEC];
  load<T, VEC>(x + c1, p);
  load<T, VEC>(x + c2, q);
  float cosine[VEC], sine[VEC];
#pragma unroll
  for (int e = 0; e < VEC; ++e) { cosine[e] = cs[e]; sine[e] = cs[half + e]; }
  if constexpr (!INTERLEAVED) {
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      const float x1 = p[e], x2 = q[e];
      p[e] = cosine[e] * x1 - sine[e] * x2;
      q[e] = sine[e] * x1 + cosine[e] * x2;
    }
  } else {
#pragma unroll
    for (int e = 0; e < VEC; ++e) {   // pair e: columns 2 e, 2 e + 1 of the 2 VEC
      float& x1 = 2 * e < VEC ? p[2 * e < VEC ? 2 * e : 0] : q[2 * e < VEC ? 0 : 2 * e - VEC];
      float& x2 = 2 * e + 1 < VEC ? p[2 * e + 1 < VEC ? 2 * e + 1 : 0] : q[2 * e + 1 < VEC ? 0 : 2 * e + 1 - VEC];
      const float y1 = cosine[e] * x1 - sine[e] * x2, y2 = sine[e] * x1 + cosine[e] * x2;
      x1 = y1;
      x2 = y2;
    }
  }
  store<T, VEC>(y + c1, p);
  store<T, VEC>(y + c2, q);
}

template <typename T, int VEC, bool INTERLEAVED>
__global__ __launch_bounds__(256) void rotary_kernel(const RotaryArgs a) {
  extern __shared__ __attribute__((aligned(16))) float table[];   // of each token: R/2 cosines, R/2 sines
  const int half = a.R / 2, tid = threadIdx.x;
  const int64_t token0 = (int64_t)blockIdx.x * a.per_group;
  const int n_tokens = a.tokens - token0 < a.per_group ? (int)(a.tokens - token0) : a.per_group;
  for (int i = tid; i < n_tokens * half; i += 256) {
    const int t = i / half, f = i % half;
    const int64_t token = token0 + t, b = token / a.S, s = token % a.S;
    int64_t p = s;
    if (a.positions) {
      const int64_t at = b * a.pos_sb + s * a.pos_ss;
      p = a.pos_is_32 ? (int64_t)reinterpret_cast<const int32_t*>(a.positions)[at] : reinterpret_cast<const int64_t*>(a.positions)[at];
    }
    double c, sn;
    cos_sin((double)p * a.inv_freq[f], c, sn);
    table[t * a.R + f] = (float)(c * a.cos_factor);
    table[t * a.R + half + f] = (float)(sn * a.sin_factor);
  }
  __shared__ int place[2 * ROTARY_TOKENS];   // of each token: its batch, its row
  if (tid < n_tokens) {
    place[2 * tid] = (int)((token0 + tid) / a.S);
    place[2 * tid + 1] = (int)((token0 + tid) % a.S);
  }
  __syncthreads();
  const int turned = half / VEC, passed = (a.D - a.R + 2 * VEC - 1) / (2 * VEC), units = turned + passed;   // of a head
  const int head0 = (int)blockIdx.y * a.heads_each, heads = a.Hq + a.Hk - head0 < a.heads_each ? a.Hq + a.Hk - head0 : a.heads_each;
  const int step_u = 256 % units, step_h = 256 / units;
  int u = tid % units, h0 = tid / units, t = 0;   // this thread's unit, head, token; 256 units on without a division
  for (;;) {
    while (h0 >= heads) {
      h0 -= heads;
      ++t;
    }
    if (t >= n_tokens) break;
    const int h = head0 + h0;
    const bool is_q = h < a.Hq;
    const RotaryOperand& o = is_q ? a.q : a.k;
    const int64_t b = place[2 * t], s = place[2 * t + 1], head = is_q ? h : h - a.Hq;
    const T* x = reinterpret_cast<const T*>(o.x) + b * o.x_sb + head * o.x_sh + s * o.x_ss;
    T* y = reinterpret_cast<T*>(o.y) + b * o.y_sb + head * o.y_sh + s * o.y_ss;
    rotate_unit<T, VEC, INTERLEAVED>(x, y, table + t * a.R, half, a.R, a.D, u, turned);
    u += step_u;
    h0 += step_h;
    if (u >= units) {
      u -= units;
      ++h0;
    }
  }
}

template <typename T, bool INTERLEAVED>
void launch(const RotaryArgs& a, int vec, dim3 grid, size_t lds, hipStream_t st) {
  switch (vec) {
    case 8:
      if constexpr (sizeof(T) == 2) { hipLaunchKernelGGL((rotary_kernel<T, 8, INTERLEAVED>), grid, dim3(256), lds, st, a); return; }
      [[fallthrough]];
    case 4: hipLaunchKernelGGL((rotary_kernel<T, 4, INTERLEAVED>), grid, dim3(256), lds, st, a); return;
    case 2: hipLaunchKernelGGL((rotary_kernel<T, 2, INTERLEAVED>), grid, dim3(256), lds, st, a); return;
    default: hipLaunchKernelGGL((rotary_kernel<T, 1, INTERLEAVED>), grid, dim3(256), lds, st, a); return;
  }
}

}  // namespace

static int rotary(const alto_mxfp4_rotary_t& p, hipStream_t st) {
  const bool has_k = p.Hk > 0;
  ALTO_REQUIRE(p.dtype == ALTO_DT_BF16 || p.dtype == ALTO_DT_F32, "rotary: dtype %d is neither bf16 (0) nor f32 (1)", p.dtype);
  ALTO_REQUIRE(p.B >= 0 && p.S >= 0 && p.Hq > 0 && p.Hk >= 0, "rotary: negative size or no query heads");
  ALTO_REQUIRE(p.D > 0 && p.R > 0 && p.R % 2 == 0 && p.R <= p.D && p.R <= 2048, "rotary: R=%lld must be even, positive, at most D=%lld and 2048", (long long)p.R, (long long)p.D);
  ALTO_REQUIRE(p.D < (1ll << 20) && p.Hq < (1ll << 20) && p.Hk < (1ll << 20) && p.B < (1ll << 31) && p.S < (1ll << 31) && product_below(1ll << 40, p.B, p.S), "rotary: size out of range");
  if (p.B == 0 || p.S == 0) return ALTO_MXFP4_OK;
  ALTO_REQUIRE(p.q && p.q_out && p.inv_freq && (!has_k || (p.k && p.k_out)), "rotary: null pointer");
  const int64_t size = p.dtype == ALTO_DT_BF16 ? 2 : 4;
  int64_t vec = 16 / size;   // elements of one access: what divides every address and the columns of either kind
  auto fits = [&](int64_t v) {
    if (p.R / 2 % v != 0 || (p.D - p.R) % v != 0) return false;
    if (((uintptr_t)p.q | (uintptr_t)p.q_out | (has_k ? (uintptr_t)p.k | (uintptr_t)p.k_out : 0)) % (uintptr_t)(v * size) != 0) return false;
    const int64_t strides[] = {p.q_sb, p.q_sh, p.q_ss, p.qo_sb, p.qo_sh, p.qo_ss, p.k_sb, p.k_sh, p.k_ss, p.ko_sb, p.ko_sh, p.ko_ss};
    for (int i = 0; i < (has_k ? 12 : 6); ++i)
      if (strides[i] % v != 0) return false;
    return true;
  };
  const int64_t strides[] = {p.q_sb, p.q_sh, p.q_ss, p.qo_sb, p.qo_sh, p.qo_ss, p.k_sb, p.k_sh, p.k_ss, p.ko_sb, p.ko_sh, p.ko_ss, p.pos_sb, p.pos_ss};
  for (const int64_t s : strides) ALTO_REQUIRE(s >= 0 && s < (1ll << 40), "rotary: strides must be non-negative");
  ALTO_REQUIRE(((uintptr_t)p.q | (uintptr_t)p.q_out | (uintptr_t)p.k | (uintptr_t)p.k_out) % (uintptr_t)size == 0 && (uintptr_t)p.inv_freq % 8 == 0 &&
                   (uintptr_t)p.positions % (p.positions_are_32 ? 4 : 8) == 0, "rotary: pointers must be aligned to their elements");
  while (vec > 1 && !fits(vec)) vec /= 2;
  RotaryArgs a{};
  a.q = {p.q, p.q_out, p.q_sb, p.q_sh, p.q_ss, p.qo_sb, p.qo_sh, p.qo_ss};
  a.k = {p.k, p.k_out, p.k_sb, p.k_sh, p.k_ss, p.ko_sb, p.ko_sh, p.ko_ss};
  a.inv_freq = p.inv_freq; a.positions = p.positions; a.pos_sb = p.pos_sb; a.pos_ss = p.pos_ss; a.pos_is_32 = p.positions_are_32 ? 1 : 0;
  a.cos_factor = p.factor;
  a.sin_factor = p.inverse ? -p.factor : p.factor;
  a.tokens = p.B * p.S; a.S = (int)p.S; a.Hq = (int)p.Hq; a.Hk = (int)p.Hk; a.D = (int)p.D; a.R = (int)p.R;
  // A workgroup has work for all threads several times over where there are tokens enough to fill the chip, else the heads of a token are spread.
  const int64_t units = (p.Hq + p.Hk) * (p.R / 2 / vec + (p.D - p.R + 2 * vec - 1) / (2 * vec));
  a.per_group = 1;
  while (a.per_group < ROTARY_TOKENS && a.per_group * units < 2048 && a.tokens / (2 * a.per_group) >= 1024 && 2 * a.per_group * p.R <= 8192) a.per_group *= 2;
  int64_t split = 1;
  while (split * a.tokens < 256 && units > 256 * split && split < p.Hq + p.Hk) split *= 2;
  a.heads_each = (int)((p.Hq + p.Hk + split - 1) / split);
  const int64_t groups = (a.tokens + a.per_group - 1) / a.per_group;
  ALTO_REQUIRE(groups < (1ll << 24), "rotary: too many tokens for one launch");   // (its threads, 256 a workgroup, are counted in 32 bits)
  const dim3 grid((unsigned)groups, (unsigned)((p.Hq + p.Hk + a.heads_each - 1) / a.heads_each));
  const size_t lds = (size_t)a.per_group * p.R * 4;
  if (p.dtype == ALTO_DT_BF16) p.interleaved ? launch<__bf16, true>(a, (int)vec, grid, lds, st) : launch<__bf16, false>(a, (int)vec, grid, lds, st);
  else p.interleaved ? launch<float, true>(a, (int)vec, grid, lds, st) : launch<float, false>(a, (int)vec, grid, lds, st);
  return check_launch("rotary");
}

}  // namespace alto

extern "C" int alto_mxfp4_rotary(const alto_mxfp4_rotary_t* p, void* stream) {
  ALTO_REQUIRE(p, "rotary: null pointer");
  return alto::rotary(*p, (hipStream_t)stream);
}
