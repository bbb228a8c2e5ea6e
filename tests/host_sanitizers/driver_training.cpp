// Host code of the entries that take their arguments as a struct (attention backward, rotary positions) under AddressSanitizer and
// UndefinedBehaviorSanitizer, without a GPU: every call fails its checks or fails at the launch, with an error code and a message.
// Each entry has valid argument sets; a call replaces zero to three of their members by plausible and extreme values.
#include <cstdint>
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <new>

#include "alto_mxfp4.h"

static bool g_no_memory = false;
void* operator new(std::size_t n) {
  void* p = g_no_memory ? nullptr : std::malloc(n ? n : 1);
  if (p == nullptr) throw std::bad_alloc();
  return p;
}
void* operator new(std::size_t n, const std::nothrow_t&) noexcept { return g_no_memory ? nullptr : std::malloc(n ? n : 1); }
void* operator new[](std::size_t n) { return operator new(n); }
void* operator new[](std::size_t n, const std::nothrow_t& t) noexcept { return operator new(n, t); }
void operator delete(void* p) noexcept { std::free(p); }
void operator delete(void* p, std::size_t) noexcept { std::free(p); }
void operator delete[](void* p) noexcept { std::free(p); }
void operator delete[](void* p, std::size_t) noexcept { std::free(p); }

namespace {

uint64_t g_state = 0x243F6A8885A308D3ull;
uint64_t next_u64() {   // splitmix64
  uint64_t z = (g_state += 0x9E3779B97F4A7C15ull);
  z = (z ^ (z >> 30)) * 0xBF58476D1CE4E5B9ull;
  z = (z ^ (z >> 27)) * 0x94D049BB133111EBull;
  return z ^ (z >> 31);
}
const int64_t kSizes[] = {-1, 0, 1, 2, 8, 31, 32, 33, 64, 96, 128, 192, 256, 1024, 8192, 65536, (1ll << 23), (1ll << 31) - 32, (1ll << 31), (1ll << 33), (1ll << 40), (1ll << 62), INT64_MAX, INT64_MIN};
const int kInts[] = {-1, 0, 1, 2, 3, 7, 130, 65536, INT32_MAX, INT32_MIN};
alignas(256) unsigned char g_mem[4096];   // stands in for device memory: the host code must never touch it
void* pool_ptr() {
  switch (next_u64() & 3) {
    case 0: return nullptr;
    case 1: return g_mem + 1;
    case 2: return g_mem + 4;
    default: return g_mem + 512;
  }
}
template <typename T, unsigned N>
T pick(const T (&pool)[N]) { return pool[next_u64() % N]; }

// sequence boundaries for 256 query tokens and 288 keys, for 4160 of either, and broken ones
struct Boundaries {
  int n;
  int32_t q[132], k[132];
};
Boundaries g_bounds[] = {{2, {0, 96, 256}, {0, 128, 288}}, {130, {}, {}}, {2, {32, 96, 256}, {0, 128, 288}}, {2, {0, 96, 224}, {0, 128, 288}}, {3, {0, 160, 96, 256}, {0, 128, 160, 288}},
                         {2, {0, 100, 256}, {0, 128, 288}}, {2, {0, INT32_MIN, 256}, {0, 128, 288}}, {2, {0, 128, 256}, {0, 96, 288}}, {2, {0, 96, 256}, {0, INT32_MAX, 288}}};

alto_mxfp4_attention_bwd_t attention(const Boundaries* b) {
  alto_mxfp4_attention_bwd_t a{};
  void* const d = g_mem + 256;
  a.q_codes = a.q_scales = a.k_codes = a.k_scales = a.vt_codes = a.v_scales = a.dout = a.out = d;
  a.lse = (const float*)d;
  a.dq = a.dk = a.dv = a.workspace = d;
  a.workspace_bytes = 1ll << 40;
  a.B = 1; a.Hq = 4; a.Hk = 2; a.Sq = 256; a.Sk = 288; a.Sk_used = 288; a.D = 128; a.Dv = 64;
  a.causal = 1; a.sm_scale = 0.1f;
  if (b) {
    a.cu_q = b->q; a.cu_k = b->k; a.n_seqs = b->n;
    if (b->n == 130) a.Sq = a.Sk = a.Sk_used = 4160;
  }
  return a;
}
void mutate(alto_mxfp4_attention_bwd_t& a) {
  const void** const p[] = {&a.q_codes, &a.k_codes, &a.vt_codes, &a.dout, &a.out, &a.k_scales};
  void** const o[] = {&a.dq, &a.dk, &a.dv, &a.workspace};
  int64_t* const s[] = {&a.workspace_bytes, &a.B, &a.Hq, &a.Hk, &a.Sq, &a.Sk, &a.Sk_used, &a.D, &a.Dv, &a.dout_sb, &a.dout_ss, &a.out_sh, &a.lse_ss, &a.dq_sb, &a.dk_sh, &a.dv_ss, &a.bias_sm, &a.alibi_sb};
  switch (next_u64() % 6) {
    case 0: *p[next_u64() % 6] = pool_ptr(); break;
    case 1: *o[next_u64() % 4] = pool_ptr(); break;
    case 2: a.bias = (const float*)pool_ptr(); a.alibi_slopes = (const float*)pool_ptr(); break;
    case 3: { const int i = pick(kInts); if (a.n_seqs == 0 || i <= 0) a.causal = i; break; }
    case 4: { const float f[] = {0.0f, -1.0f, 1e30f, __builtin_nanf(""), __builtin_inff()}; a.sm_scale = pick(f); break; }
    default: *s[next_u64() % 18] = pick(kSizes); break;
  }
}
alto_mxfp4_rotary_t rotary() {
  alto_mxfp4_rotary_t a{};
  a.q = a.k = a.q_out = a.k_out = g_mem + 256;
  a.inv_freq = (const double*)(g_mem + 256);
  a.B = 2; a.S = 100; a.Hq = 4; a.Hk = 2; a.D = 128; a.R = 64; a.factor = 1.0;
  return a;
}
void mutate(alto_mxfp4_rotary_t& a) {
  const void** const p[] = {&a.q, &a.k, &a.positions};
  int64_t* const s[] = {&a.B, &a.S, &a.Hq, &a.Hk, &a.D, &a.R, &a.q_sb, &a.q_sh, &a.q_ss, &a.k_sb, &a.qo_ss, &a.ko_sh, &a.pos_sb, &a.pos_ss};
  switch (next_u64() % 4) {
    case 0: *p[next_u64() % 3] = pool_ptr(); break;
    case 1: a.q_out = pool_ptr(); break;
    case 2: a.dtype = pick(kInts); a.positions_are_32 = pick(kInts); break;
    default: *s[next_u64() % 14] = pick(kSizes); break;
  }
}

struct Count {
  long calls = 0, ok = 0, launches = 0;
};
bool looked_at(Count& c, int64_t rc, const char* what) {
  ++c.calls;
  if (rc >= 0) { ++c.ok; return true; }
  const char* msg = alto_mxfp4_last_error();
  if (msg == nullptr || std::strlen(msg) == 0) {
    std::fprintf(stderr, "%s: error code %lld without a message\n", what, (long long)rc);
    return false;
  }
  if (std::strstr(msg, "launch failed") != nullptr || std::strstr(msg, "could not reserve") != nullptr) ++c.launches;
  return true;
}

}  // namespace

int main(int argc, char** argv) {
  const long rounds = argc > 1 ? std::atol(argv[1]) : 2000;
  for (int k = 0; k <= 130; ++k) g_bounds[1].q[k] = g_bounds[1].k[k] = 32 * k;
  Count bwd, size, rot;
  for (long it = 0; it < rounds; ++it) {
    const unsigned which = next_u64() % (2 * sizeof(g_bounds) / sizeof(g_bounds[0]));
    alto_mxfp4_attention_bwd_t a = attention(which < sizeof(g_bounds) / sizeof(g_bounds[0]) ? &g_bounds[which] : nullptr);
    for (int c = (int)(next_u64() % 4); c > 0; --c) mutate(a);
    if (!looked_at(bwd, alto_mxfp4_attention_bwd(&a, nullptr), "attention_bwd") || !looked_at(size, alto_mxfp4_attention_bwd_workspace_bytes(&a), "attention_bwd_workspace_bytes")) return 2;
    alto_mxfp4_rotary_t r = rotary();
    for (int c = (int)(next_u64() % 4); c > 0; --c) mutate(r);
    if (!looked_at(rot, alto_mxfp4_rotary(&r, nullptr), "rotary")) return 2;
  }
  if (alto_mxfp4_attention_bwd(nullptr, nullptr) != -1 || alto_mxfp4_attention_bwd_workspace_bytes(nullptr) != -1 || alto_mxfp4_rotary(nullptr, nullptr) != -1) return 3;
  alto_mxfp4_attention_bwd_t a = attention(&g_bounds[0]);
  g_no_memory = true;
  const int rc = alto_mxfp4_attention_bwd(&a, nullptr);
  g_no_memory = false;
  if (rc >= 0 || std::strstr(alto_mxfp4_last_error(), "memory") == nullptr) {
    std::fprintf(stderr, "attention_bwd without host memory: code %d, %s\n", rc, alto_mxfp4_last_error());
    return 5;
  }
  for (unsigned k = 0; k < sizeof(g_mem); ++k)
    if (g_mem[k] != 0) {
      std::fprintf(stderr, "host code wrote through a pointer that stands for device memory (byte %u)\n", k);
      return 3;
    }
  std::printf("attention_bwd calls %ld launches %ld\nworkspace calls %ld answers %ld\nrotary calls %ld launches %ld\n", bwd.calls, bwd.launches, size.calls, size.ok, rot.calls, rot.launches);
  return rounds >= 100 && (bwd.launches == 0 || size.ok == 0 || rot.launches == 0) ? 4 : 0;
}
