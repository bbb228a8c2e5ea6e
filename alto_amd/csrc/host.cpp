// Host side of the entry points in one native call each: output tensors, argument checks and the launch through the C ABI
// (include/alto_mxfp4.h), as a CPython module that alto_amd/_lib.py loads beside the kernel library.
//
// Per call the Python form of the same work cost 24 us (quantizer: four torch.empty, views, a 29-argument ctypes call),
// 10 us (GEMM) and 19 us (Hadamard draw) against 3 us for the launch itself, which is most of a training step of a small
// layer and all of a decode step; here they cost 8, 4 and 5 us, launch included.
//
// Every function either serves the call or declines it (returns None) before it has done anything; the Python caller then
// goes on with the general path, which also words the errors.  The kernel library is reached through the function addresses
// that `bind` is given, so that there is one library per process whichever file it came from.
#include <pybind11/stl.h>
#include <torch/csrc/utils/pybind.h>

#include <ATen/ATen.h>
#include <c10/core/impl/LocalDispatchKeySet.h>
#include <c10/hip/HIPFunctions.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/python_cpp_function.h>

#include <algorithm>
#include <cstring>
#include <optional>
#include <string>
#include <vector>

#include "../../include/alto_mxfp4.h"

namespace py = pybind11;
using at::Tensor;
using OptTensor = std::optional<Tensor>;

namespace {

struct Api {
#define ALTO_FN(name) decltype(&alto_mxfp4_##name) name = nullptr
  ALTO_FN(quantize_ex);
  ALTO_FN(quantize_sr_hw);
  ALTO_FN(quantize_sr_hw_words);
  ALTO_FN(philox_advance);
  ALTO_FN(dequantize);
  ALTO_FN(gemm);
  ALTO_FN(gemm_ps);
  ALTO_FN(grouped_gemm_ps);
  ALTO_FN(grouped_gemm_workspace_bytes);
  ALTO_FN(grouped_gemm_dw_ps);
  ALTO_FN(grouped_gradients_ps);
  ALTO_FN(attention_quantize);
  ALTO_FN(attention_fwd_strided);
  ALTO_FN(attention_quantize_kv);
  ALTO_FN(attention_fwd_bf16q);
  ALTO_FN(grouped_gemm_plan_ends);
  ALTO_FN(quantize_operands);
  ALTO_FN(gemm_two);
  ALTO_FN(attention_bwd);
  ALTO_FN(attention_bwd_workspace_bytes);
  ALTO_FN(rotary);
  ALTO_FN(fp8_token_blocks);
  ALTO_FN(fp8_quantize);
  ALTO_FN(fp8_gemm);
  ALTO_FN(fp8_grouped_gemm);
  ALTO_FN(fp8_grouped_gemm_weights);
#undef ALTO_FN
} api;
py::object* check_fn = nullptr;   // _lib.check(rc, name): raises for rc != 0 (never freed: the interpreter may be gone by then)

void bind(const py::dict& address, py::object check) {
#define ALTO_FN(name) api.name = reinterpret_cast<decltype(api.name)>(address["alto_mxfp4_" #name].cast<uintptr_t>())
  ALTO_FN(quantize_ex);
  ALTO_FN(quantize_sr_hw);
  ALTO_FN(quantize_sr_hw_words);
  ALTO_FN(philox_advance);
  ALTO_FN(dequantize);
  ALTO_FN(gemm);
  ALTO_FN(gemm_ps);
  ALTO_FN(grouped_gemm_ps);
  ALTO_FN(grouped_gemm_workspace_bytes);
  ALTO_FN(grouped_gemm_dw_ps);
  ALTO_FN(grouped_gradients_ps);
  ALTO_FN(attention_quantize);
  ALTO_FN(attention_fwd_strided);
  ALTO_FN(attention_quantize_kv);
  ALTO_FN(attention_fwd_bf16q);
  ALTO_FN(grouped_gemm_plan_ends);
  ALTO_FN(quantize_operands);
  ALTO_FN(gemm_two);
  ALTO_FN(attention_bwd);
  ALTO_FN(attention_bwd_workspace_bytes);
  ALTO_FN(rotary);
  ALTO_FN(fp8_token_blocks);
  ALTO_FN(fp8_quantize);
  ALTO_FN(fp8_gemm);
  ALTO_FN(fp8_grouped_gemm);
  ALTO_FN(fp8_grouped_gemm_weights);
#undef ALTO_FN
  delete check_fn;
  check_fn = new py::object(std::move(check));
}

// the launch without the interpreter lock, as ctypes makes it; a refused call raises what _lib.check makes of it
template <typename F, typename... A>
void call(const char* name, F fn, A... args) {
  int rc;
  {
    py::gil_scoped_release nogil;
    rc = fn(args...);
  }
  if (rc != 0) (*check_fn)(rc, name);
}

int dtype_code(at::ScalarType t) { return t == at::kBFloat16 ? ALTO_DT_BF16 : ALTO_DT_F32; }
bool is_float(const Tensor& t) { return t.scalar_type() == at::kBFloat16 || t.scalar_type() == at::kFloat; }
// (a wrapper subclass has no storage of its own: the Python route resolves it)
bool on_gpu(const Tensor& t) { return t.is_cuda() && t.layout() == at::kStrided && !t.unsafeGetTensorImpl()->is_python_dispatch(); }
uint8_t* bytes(const Tensor& t) { return t.defined() ? static_cast<uint8_t*>(t.data_ptr()) : nullptr; }
bool aligned16(const Tensor& t) { return (reinterpret_cast<uintptr_t>(t.data_ptr()) & 15) == 0; }
int64_t stride_of(const Tensor& t, int64_t d) { return t.size(d) == 1 ? 0 : t.stride(d); }   // a dim of one is never stepped over: its stride may be anything
int64_t div_up(int64_t a, int64_t b) { return (a + b - 1) / b; }
// attention.py:_readable.  (contiguous() would hand back a dense tensor at an odd address as it is)
Tensor readable_rows(const Tensor& t) {
  const int64_t vec = 16 / t.element_size();
  return t.stride(3) == 1 && aligned16(t) && stride_of(t, 0) % vec == 0 && stride_of(t, 1) % vec == 0 && stride_of(t, 2) % vec == 0 ? t : t.clone(at::MemoryFormat::Contiguous);
}

// (torch.jit.trace would record the outputs' allocation and none of the launches: the general functions end in an error there)
bool being_traced() { return c10::impl::tls_is_dispatch_key_included(c10::DispatchKey::Tracer); }
// A call that a node may serve: not under torch.jit.trace, a functorch transform or forward-mode differentiation, which the general
// functions refuse
bool node_serves(const Tensor& x, const Tensor& weight) {
  return !being_traced() && !c10::impl::tls_is_dispatch_key_included(c10::DispatchKey::FuncTorchDynamicLayerFrontMode) && !x._fw_grad(0).defined() &&
         !weight._fw_grad(0).defined();
}

struct Alloc {
  at::TensorOptions u8;
  explicit Alloc(const Tensor& like) : u8(at::TensorOptions().dtype(at::kByte).device(like.device())) {}
  Tensor dense(at::IntArrayRef size) const { return at::empty(size, u8); }
  // [R, n] (flat) or [B, R, n] codes, rows on 128-byte boundaries with pad; transposed: the flat view [n, R]
  Tensor codes(int64_t B, int64_t R, int64_t n, bool pad, bool flat, bool transposed) const {
    const int64_t pitch = pad ? div_up(n, 128) * 128 : n;
    if (flat && transposed) return at::empty_strided({n, R}, {1, pitch}, u8);
    if (flat) return at::empty_strided({R, n}, {pitch, 1}, u8);
    return at::empty_strided({B, R, n}, {R * pitch, pitch, 1}, u8);
  }
};

// quantization.py:_quantize_call.  x [B, M, C] or, with flat, [M, C]; flat: the outputs come as quantize_rowcol returns them
// (column codes and plain column scales as transposed views).
py::object quantize(const Tensor& x_in, bool flat, bool want_row, bool want_col, bool is_2d, int sr_mode, const OptTensor& rand, uint64_t seed, uint64_t offset,
                    const OptTensor& state, const OptTensor& signs, const OptTensor& perm, int clip, bool uos, bool pad, bool pack_row, bool pack_col,
                    uintptr_t stream) {
  Tensor x = x_in;
  if (!on_gpu(x) || !is_float(x) || x.dim() != (flat ? 2 : 3)) return py::none();
  const int64_t vec = x.scalar_type() == at::kBFloat16 ? 8 : 4;
  auto readable = [&](const Tensor& t) {   // unit stride along C, everything else in whole 16-byte units
    if (t.stride(-1) != 1 || !aligned16(t)) return false;
    for (int64_t d = 0; d + 1 < t.dim(); ++d)
      if (stride_of(t, d) % vec != 0) return false;
    return true;
  };
  if (!readable(x)) {
    if (!flat) return py::none();
    x = x.contiguous();
    if (!readable(x)) return py::none();
  }
  const int64_t B = flat ? 1 : x.size(0), M = x.size(-2), C = x.size(-1);
  const int64_t ld_x = M > 1 ? x.stride(-2) : C, bs_x = B > 1 ? x.stride(0) : M * ld_x;
  int64_t ld_r = 0, bs_r = 0;
  const uint32_t* words = nullptr;
  if (rand.has_value()) {
    if (!on_gpu(*rand) || rand->dim() != 3) return py::none();
    ld_r = M > 1 ? rand->stride(1) : C;
    bs_r = B > 1 ? rand->stride(0) : M * ld_r;
    words = static_cast<const uint32_t*>(rand->data_ptr());
  }
  const Alloc a(x);
  Tensor rc, rs, cc, cs;
  if (want_row) {
    rc = a.codes(B, M, C / 2, pad, flat, false);
    if (pack_row) rs = flat ? a.dense({div_up(C / 32, 16), M, 16}) : a.dense({B, div_up(C / 32, 16), M, 16});
    else rs = flat ? a.dense({is_2d ? M / 32 : M, C / 32}) : a.dense({B, is_2d ? M / 32 : M, C / 32});
  }
  if (want_col) {
    cc = a.codes(B, C, M / 2, pad, flat, true);
    const int64_t rows = is_2d ? C / 32 : C;
    if (pack_col) cs = flat ? a.dense({div_up(M / 32, 16), C, 16}) : a.dense({B, div_up(M / 32, 16), C, 16});
    else cs = flat ? at::empty_strided({M / 32, rows}, {1, M / 32}, a.u8) : a.dense({B, rows, M / 32});
  }
  const int64_t ld_rc = want_row ? rc.stride(-2) : 0, ld_cc = want_col ? cc.stride(flat ? 1 : -2) : 0;
  const int dt = dtype_code(x.scalar_type()), had = signs.has_value();
  const int8_t* sp = had ? static_cast<const int8_t*>(signs->data_ptr()) : nullptr;
  const uint8_t* pp = perm.has_value() ? static_cast<const uint8_t*>(perm->data_ptr()) : nullptr;
  const uint64_t* st = state.has_value() ? static_cast<const uint64_t*>(state->data_ptr()) : nullptr;
  void* s = reinterpret_cast<void*>(stream);
  if (sr_mode == 3 && !pack_row && !pack_col)
    call("alto_mxfp4_quantize_sr_hw", api.quantize_sr_hw, x.data_ptr(), dt, B, M, C, ld_x, bs_x, bytes(rc), bytes(rs), bytes(cc), bytes(cs), ld_rc, ld_cc, (int)is_2d,
         seed, offset, st, had, sp, pp, clip, (int)uos, s);
  else
    call("alto_mxfp4_quantize_ex", api.quantize_ex, x.data_ptr(), dt, B, M, C, ld_x, bs_x, bytes(rc), bytes(rs), bytes(cc), bytes(cs), ld_rc, ld_cc, (int)is_2d, sr_mode,
         words, ld_r, bs_r, seed, offset, st, had, sp, pp, clip, (int)uos, (pack_row ? ALTO_QUANT_PACK_ROW_SCALES : 0) | (pack_col ? ALTO_QUANT_PACK_COL_SCALES : 0), s);
  if (st != nullptr)
    call("alto_mxfp4_philox_advance", api.philox_advance, static_cast<uint64_t*>(state->data_ptr()),
         (uint64_t)(sr_mode == 3 ? api.quantize_sr_hw_words(dt, B, M, C) : B * M * C), s);
  auto opt = [](const Tensor& t) -> py::object { return t.defined() ? py::cast(t) : py::none(); };
  return py::make_tuple(opt(rc), opt(rs), opt(cc), opt(cs));
}

// quantization.py:convert_from_mxfp4 of a 2D tensor
py::object dequantize(const Tensor& codes, const Tensor& scales, bool f32, bool last_axis, bool is_2d, int clip, uintptr_t stream) {
  if (!on_gpu(codes) || !on_gpu(scales) || codes.dim() != 2 || scales.dim() != 2 || codes.scalar_type() != at::kByte || scales.scalar_type() != at::kByte) return py::none();
  const int64_t R = codes.size(last_axis ? 0 : 1), C = 2 * codes.size(last_axis ? 1 : 0);
  if (R == 0 || C == 0 || C % 32 != 0 || (is_2d && R % 32 != 0)) return py::none();
  if (scales.size(last_axis ? 0 : 1) != (is_2d ? R / 32 : R) || scales.size(last_axis ? 1 : 0) != C / 32) return py::none();
  const Tensor l = (last_axis ? codes : codes.t()).contiguous(), sc = (last_axis ? scales : scales.t()).contiguous();
  const Tensor out = at::empty({R, C}, at::TensorOptions().dtype(f32 ? at::kFloat : at::kBFloat16).device(codes.device()));
  call("alto_mxfp4_dequantize", api.dequantize, bytes(l), bytes(sc), R, C, (int)is_2d, out.data_ptr(), f32 ? ALTO_DT_F32 : ALTO_DT_BF16, C, (int64_t)1, clip,
       reinterpret_cast<void*>(stream));
  return py::cast(last_axis ? out : out.t());
}

// linear.py:blockwise_mxfp4_gemm with both operands packed along K
py::object gemm(const Tensor& a_in, const Tensor& as_in, const Tensor& b_in, const Tensor& bs_in, bool a_2d, bool b_2d, bool trans_a, bool trans_b, bool f32,
                double out_scale, uintptr_t stream) {
  for (const Tensor* t : {&a_in, &as_in, &b_in, &bs_in})
    if (!on_gpu(*t) || t->dim() != 2 || t->scalar_type() != at::kByte) return py::none();
  // codes [rows, K/2], scales [rows (/32), K/32], as sizes and strides of the tensors as given
  const int ar = trans_a ? 1 : 0, ak = 1 - ar, br = trans_b ? 0 : 1, bk = 1 - br;
  const int64_t M = a_in.size(ar), K = 2 * a_in.size(ak), N = b_in.size(br);
  if (M == 0 || N == 0 || K == 0 || K % 32 != 0 || 2 * b_in.size(bk) != K || (a_2d && M % 32 != 0) || (b_2d && N % 32 != 0)) return py::none();
  if (as_in.size(ar) != (a_2d ? M / 32 : M) || as_in.size(ak) != K / 32 || bs_in.size(br) != (b_2d ? N / 32 : N) || bs_in.size(bk) != K / 32) return py::none();
  if (a_in.stride(ak) != 1 || a_in.stride(ar) % 16 != 0 || !aligned16(a_in) || b_in.stride(bk) != 1 || b_in.stride(br) % 16 != 0 || !aligned16(b_in)) return py::none();
  const Tensor c = at::empty({M, N}, at::TensorOptions().dtype(f32 ? at::kFloat : at::kBFloat16).device(a_in.device()));
  call("alto_mxfp4_gemm", api.gemm, bytes(a_in), a_in.stride(ar), bytes(as_in), as_in.stride(ar), as_in.stride(ak), (int)a_2d, bytes(b_in), b_in.stride(br), bytes(bs_in),
       bs_in.stride(br), bs_in.stride(bk), (int)b_2d, M, N, K, c.data_ptr(), f32 ? ALTO_DT_F32 : ALTO_DT_BF16, N, (float)out_scale, reinterpret_cast<void*>(stream));
  return py::cast(c);
}

bool packed_scales(const Tensor& t, int64_t K, int64_t rows) {
  return on_gpu(t) && t.scalar_type() == at::kByte && t.dim() == 3 && t.size(0) == div_up(K / 32, 16) && t.size(1) == rows && t.size(2) == 16 && t.is_contiguous();
}

// linear.py:gemm_packed
py::object gemm_packed(const Tensor& a, const Tensor& a_ps, const Tensor& b, const Tensor& b_ps, double out_scale, uintptr_t stream) {
  if (!on_gpu(a) || !on_gpu(b) || a.dim() != 2 || b.dim() != 2 || a.stride(1) != 1 || b.stride(1) != 1 || a.size(1) != b.size(1)) return py::none();
  const int64_t M = a.size(0), N = b.size(0), K = 2 * a.size(1);
  if (!packed_scales(a_ps, K, M) || !packed_scales(b_ps, K, N)) return py::none();
  const Tensor c = at::empty({M, N}, at::TensorOptions().dtype(at::kBFloat16).device(a.device()));
  call("alto_mxfp4_gemm_ps", api.gemm_ps, bytes(a), a.stride(0), bytes(a_ps), bytes(b), b.stride(0), bytes(b_ps), M, N, K, c.data_ptr(), N, (float)out_scale,
       reinterpret_cast<void*>(stream));
  return py::cast(c);
}

// grouped_gemm.py:grouped_forward_packed -> (out, pass list)
py::object grouped_packed(const Tensor& a, const Tensor& a_ps, const Tensor& w, const Tensor& w_ps, const Tensor& offs, const OptTensor& expert, int n_groups,
                          const OptTensor& plan, uintptr_t stream) {
  if (!on_gpu(a) || !on_gpu(w) || !on_gpu(offs) || a.dim() != 2 || w.dim() != 3 || a.stride(1) != 1 || w.stride(2) != 1 || a.size(1) != w.size(2)) return py::none();
  const int64_t E = w.size(0), N = w.size(1), M = a.size(0), K = 2 * a.size(1), KB = div_up(K / 32, 16);
  if (!packed_scales(a_ps, K, M) || !on_gpu(w_ps) || w_ps.dim() != 4 || w_ps.size(0) != E || w_ps.size(1) != KB || w_ps.size(2) != N || w_ps.size(3) != 16 || !w_ps.is_contiguous())
    return py::none();
  const Tensor out = at::empty({M, N}, at::TensorOptions().dtype(at::kBFloat16).device(a.device()));
  const Tensor ws = plan.has_value() ? *plan : Alloc(a).dense({api.grouped_gemm_workspace_bytes(M, n_groups)});
  call("alto_mxfp4_grouped_gemm_ps", api.grouped_gemm_ps, bytes(a), a.stride(0), bytes(a_ps), bytes(w), w.stride(0), w.stride(1), bytes(w_ps), w_ps.stride(0),
       static_cast<const int32_t*>(offs.data_ptr()), expert.has_value() ? static_cast<const int32_t*>(expert->data_ptr()) : nullptr, n_groups, (int)E, M, N, K, out.data_ptr(),
       N, ws.data_ptr(), ws.numel(), (int)plan.has_value(), reinterpret_cast<void*>(stream));
  return py::make_tuple(out, ws);
}

// grouped_gemm.py:grouped_dw_packed
py::object grouped_dw_packed(const Tensor& go, const Tensor& go_ps, const Tensor& x, const Tensor& x_ps, const Tensor& offs, const OptTensor& expert, int n_groups,
                             int n_experts, bool trans_weights, double out_scale, uintptr_t stream) {
  if (!on_gpu(go) || !on_gpu(x) || !on_gpu(offs) || go.dim() != 2 || x.dim() != 2 || go.size(1) != x.size(1)) return py::none();
  if (go.stride(1) != 1 || go.stride(0) % 16 != 0 || x.stride(1) != 1 || x.stride(0) % 16 != 0) return py::none();
  const int64_t N = go.size(0), K = x.size(0), M = 2 * go.size(1);
  if (M % 32 != 0 || !packed_scales(go_ps, M, N) || !packed_scales(x_ps, M, K)) return py::none();
  const auto opts = at::TensorOptions().dtype(at::kBFloat16).device(go.device());
  const Tensor dw = trans_weights ? at::empty({n_experts, N, K}, opts) : at::empty({n_experts, K, N}, opts);
  call("alto_mxfp4_grouped_gemm_dw_ps", api.grouped_gemm_dw_ps, bytes(go), go.stride(0), bytes(go_ps), bytes(x), x.stride(0), bytes(x_ps),
       static_cast<const int32_t*>(offs.data_ptr()), expert.has_value() ? static_cast<const int32_t*>(expert->data_ptr()) : nullptr, n_groups, n_experts, M, N, K, dw.data_ptr(),
       dw.stride(0), trans_weights ? dw.stride(1) : dw.stride(2), trans_weights ? dw.stride(2) : dw.stride(1), (float)out_scale, reinterpret_cast<void*>(stream));
  return py::cast(dw);
}

// attention.py:_attend without ALiBi slopes: operand quantizer and attention kernel on [B, H, S, D] views (bf16: the attention
// kernel quantizes Q itself)
bool attend(const Tensor& q_in, const Tensor& k_in, const Tensor& v_in, double sm_scale, bool causal, const Tensor& out, const Tensor& lse,
            const std::vector<int32_t>& cu_q, const std::vector<int32_t>& cu_k, uintptr_t stream) {
  if (!node_serves(q_in, k_in) || v_in._fw_grad(0).defined()) return false;
  Tensor q = q_in, k = k_in, v = v_in;
  for (Tensor* t : {&q, &k, &v}) {
    if (!on_gpu(*t) || !is_float(*t) || t->dim() != 4 || t->scalar_type() != q_in.scalar_type()) return false;
    *t = readable_rows(*t);
  }
  const int64_t B = q.size(0), Hq = q.size(1), Sq = q.size(2), D = q.size(3), Hk = v.size(1), Sk = v.size(2), Dv = v.size(3);
  if (k.size(0) != v.size(0) || k.size(1) != Hk || k.size(2) != Sk || B != k.size(0) || k.size(3) != D) return false;
  // 16 bytes of room behind each part: the attention kernel reads K's and V's scale bytes in whole dwords
  const bool own_q = q.scalar_type() == at::kBFloat16;
  const int64_t sizes[6] = {B * Hk * Sk * D / 2, B * Hk * Sk * Dv / 2, B * Hk * (Sk / 32) * (D / 32), B * Hk * (Sk / 32) * (Dv / 32),
                            own_q ? 0 : B * Hq * Sq * D / 2, own_q ? 0 : B * Hq * (Sq / 32) * (D / 32)};
  int64_t start[6], total = 0;
  for (int i = 0; i < (own_q ? 4 : 6); ++i) {
    start[i] = total;
    total += div_up(sizes[i] + 16, 256) * 256;
  }
  const Tensor buf = Alloc(q).dense({total});
  uint8_t* p = bytes(buf);
  uint8_t *kq = p + start[0], *vq = p + start[1], *ks = p + start[2], *vs = p + start[3];
  void* s = reinterpret_cast<void*>(stream);
  const int n = cu_q.empty() ? 0 : (int)cu_q.size() - 1;
  const int32_t *cq = n ? cu_q.data() : nullptr, *ck = n ? cu_k.data() : nullptr;
  float* lse_p = static_cast<float*>(lse.data_ptr());
  if (own_q) {
    call("alto_mxfp4_attention_quantize_kv", api.attention_quantize_kv, k.data_ptr(), v.data_ptr(), (int)ALTO_DT_BF16, B, Hk, Sk, D, Dv, stride_of(k, 0), stride_of(k, 1),
         stride_of(k, 2), stride_of(v, 0), stride_of(v, 1), stride_of(v, 2), kq, ks, vq, vs, s);
    call("alto_mxfp4_attention_fwd_bf16q", api.attention_fwd_bf16q, q.data_ptr(), stride_of(q, 0), stride_of(q, 1), stride_of(q, 2), kq, ks, vq, vs, out.data_ptr(), lse_p, B,
         Hq, Hk, Sq, Sk, D, Dv, out.stride(0), out.stride(1), out.stride(2), lse.stride(0), lse.stride(1), lse.stride(2), n, cq, ck, (float)sm_scale, (int)causal, s);
    return true;
  }
  uint8_t *qq = p + start[4], *qs = p + start[5];
  call("alto_mxfp4_attention_quantize", api.attention_quantize, q.data_ptr(), k.data_ptr(), v.data_ptr(), (int)ALTO_DT_F32, B, Hq, Hk, Sq, Sk, D, Dv, stride_of(q, 0),
       stride_of(q, 1), stride_of(q, 2), stride_of(k, 0), stride_of(k, 1), stride_of(k, 2), stride_of(v, 0), stride_of(v, 1), stride_of(v, 2), qq, qs, kq, ks, vq, vs, s);
  call("alto_mxfp4_attention_fwd_strided", api.attention_fwd_strided, qq, qs, kq, ks, vq, vs, out.data_ptr(), lse_p, B, Hq, Hk, Sq, Sk, D, Dv, out.stride(0), out.stride(1),
       out.stride(2), lse.stride(0), lse.stride(1), lse.stride(2), n, cq, ck, (float)sm_scale, (int)causal, static_cast<const float*>(nullptr), (int64_t)0, (int64_t)0, s);
  return true;
}

bool on_current_device(const Tensor& t) { return on_gpu(t) && t.get_device() == c10::hip::current_device(); }

// ------------------------------------------------------------------------------------------------- whole training directions
// A layer's step as an autograd node of its own, one native call per direction: outputs, quantizers and products, the interpreter
// lock given up.  What a direction needs only itself shares one buffer, what the backward needs of either operand has one of its own.
// The backward runs on the engine's device thread while the caller waits, and every handover of the interpreter lock between the two
// is a wake-up more.  A node of its own needs the interpreter only where the gradient is rounded stochastically, to ask which source of
// random words is installed; a Python function whose two directions were native calls needed it for each.  Whole steps, five processes
// of either in turn: 512 x 1024 x 1024 110 to 114 us as that function (one process 68: how fast a waiting thread wakes differs from
// process to process), 90 to 94 as a node; 2048 x 4096 x 4096 102 to 111, 96; fp32 1376 x 2880 x 2144 94 to 97 (one 69), 78 to 83; expert
// layer of 2560 x 1024 x 1440 120 to 123, 94 to 98.  (About 40 us of a small step are the engine's own two wake-ups.)
struct Failure {
  int rc = 0;
  const char* name = "";
  bool ok(const char* what, int code) {
    if (code != 0) { rc = code; name = what; }
    return code == 0;
  }
  void raise() const {
    if (rc != 0) (*check_fn)(rc, name);
  }
};

int64_t pitch128(int64_t n) { return div_up(n, 128) * 128; }
int64_t up256(int64_t n) { return div_up(n, 256) * 256; }
int64_t packed_bytes(int64_t K, int64_t rows) { return div_up(K / 32, 16) * rows * 16; }

// One of the two copies a quantizer pass makes of `batch` matrices: codes [rows][pitch of K / 2 bytes], then scales, packed or
// [rows (/ 32)][K / 32].  Bytes of a buffer from `at` on.
struct Copy {
  int64_t rows = 0, K = 0, batch = 1, at = 0;
  bool packed = false, is_2d = false;
  int64_t ld() const { return pitch128(K / 2); }
  int64_t scale_ld() const { return K / 32; }
  int64_t scale_bytes() const { return packed ? packed_bytes(K, rows) : (is_2d ? rows / 32 : rows) * scale_ld(); }
  int64_t scales_at() const { return at + up256(batch * rows * ld()); }
  int64_t end() const { return scales_at() + up256(batch * scale_bytes() + 16); }
  uint8_t* codes(const Tensor& buf) const { return bytes(buf) + at; }
  uint8_t* scales(const Tensor& buf) const { return bytes(buf) + scales_at(); }
};

// [batch][M][C] with unit stride along C in whole 16-byte units, as `quantize` reads it
bool rows_readable(const Tensor& t) {
  if (!on_gpu(t) || !is_float(t) || t.stride(-1) != 1 || !aligned16(t)) return false;
  const int64_t vec = t.scalar_type() == at::kBFloat16 ? 8 : 4;
  for (int64_t d = 0; d + 1 < t.dim(); ++d)
    if (t.size(d) != 1 && (t.stride(d) % vec != 0 || t.stride(d) < t.size(-1))) return false;
  return true;
}

// The options of a step, by value: what its node keeps for the backward besides the saved buffers
struct StepOptions {
  bool hadamard = false, permuted = false, uos = false, sr = false, dge = false, trans_weights = false;
  int clip = 0, packed = 0;
  int64_t E = 0, N = 0, K = 0;
  double out_scale = 1.0;   // of the weight gradient
  at::ScalarType dtype = at::kFloat;
  int8_t signs[32];
  uint8_t perm[32];
  StepOptions() = default;
  // signs int8[32] and perm uint8[32] on the host, as HadamardTransform keeps them
  StepOptions(const OptTensor& s, const OptTensor& p, int clip_, bool uos_, bool sr_, bool dge_, double out_scale_) : uos(uos_), sr(sr_), dge(dge_), clip(clip_), out_scale(out_scale_) {
    hadamard = s.has_value();
    permuted = p.has_value();
    if (hadamard) std::memcpy(signs, s->data_ptr(), 32);
    if (permuted) std::memcpy(perm, p->data_ptr(), 32);
  }
};
struct Hadamard {
  int on = 0;
  const int8_t* signs = nullptr;
  const uint8_t* perm = nullptr;
  explicit Hadamard(const StepOptions& o) : on(o.hadamard), signs(o.hadamard ? o.signs : nullptr), perm(o.permuted ? o.perm : nullptr) {}
};

// both copies of a gradient [row.rows, col.rows], 1D blocks; sr_mode 0 (nearest) or 3 (the hardware's stochastic converts)
bool quantize_gradient(Failure& f, const Tensor& x, const Copy& row, const Tensor& row_buf, const Copy& col, const Tensor& col_buf, int sr_mode, uint64_t seed,
                       const Hadamard& h, int clip, bool uos, void* s) {
  const int64_t M = row.rows, C = col.rows, ld = M > 1 ? x.stride(-2) : C, bs = M * ld;
  const int dt = dtype_code(x.scalar_type());
  if (sr_mode == 3 && !row.packed && !col.packed)
    return f.ok("alto_mxfp4_quantize_sr_hw", api.quantize_sr_hw(x.data_ptr(), dt, 1, M, C, ld, bs, row.codes(row_buf), row.scales(row_buf), col.codes(col_buf),
                                                                col.scales(col_buf), row.ld(), col.ld(), 0, seed, 0, nullptr, h.on, h.signs, h.perm, clip, (int)uos, s));
  return f.ok("alto_mxfp4_quantize_ex",
              api.quantize_ex(x.data_ptr(), dt, 1, M, C, ld, bs, row.codes(row_buf), row.scales(row_buf), col.codes(col_buf), col.scales(col_buf), row.ld(), col.ld(),
                              0, sr_mode, nullptr, 0, 0, seed, 0, nullptr, h.on, h.signs, h.perm, clip, (int)uos,
                              (row.packed ? ALTO_QUANT_PACK_ROW_SCALES : 0) | (col.packed ? ALTO_QUANT_PACK_COL_SCALES : 0), s));
}

// both copies of x (1D blocks) and of W (2D blocks), round to nearest; w_row / w_col: the copies along W's columns and along its rows
bool quantize_operands(Failure& f, const Tensor& x, const Copy& x_row, const Tensor& x_row_buf, const Copy& x_col, const Tensor& x_col_buf, const Hadamard& h, int clip,
                       const Tensor& w, const Copy& w_row, const Tensor& w_row_buf, const Copy& w_col, const Tensor& w_col_buf, bool uos, void* s) {
  const int64_t M = x_row.rows, K = x_col.rows, B = w_row.batch, R = w_row.rows, C = w_col.rows, ld_w = R > 1 ? w.stride(-2) : C;
  auto flags = [](const Copy& r, const Copy& c) { return (r.packed ? ALTO_QUANT_PACK_ROW_SCALES : 0) | (c.packed ? ALTO_QUANT_PACK_COL_SCALES : 0); };
  return f.ok("alto_mxfp4_quantize_operands",
              api.quantize_operands(x.data_ptr(), dtype_code(x.scalar_type()), M, K, M > 1 ? x.stride(-2) : K, x_row.codes(x_row_buf), x_row.scales(x_row_buf),
                                    x_col.codes(x_col_buf), x_col.scales(x_col_buf), x_row.ld(), x_col.ld(), h.on, h.signs, h.perm, clip, flags(x_row, x_col), w.data_ptr(),
                                    dtype_code(w.scalar_type()), B, R, C, ld_w, B > 1 ? w.stride(0) : R * ld_w, w_row.codes(w_row_buf), w_row.scales(w_row_buf),
                                    w_col.codes(w_col_buf), w_col.scales(w_col_buf), w_row.ld(), w_col.ld(), flags(w_row, w_col), (int)uos, s));
}

alto_mxfp4_product product_of(const Copy& a, const Tensor& a_buf, const Copy& b, const Tensor& b_buf, const Tensor& c, double out_scale) {
  return {a.codes(a_buf), a.scales(a_buf), b.codes(b_buf), b.scales(b_buf), a.ld(), a.scale_ld(), 1, b.ld(), b.scale_ld(), 1, a.rows, b.rows, a.K, c.data_ptr(), b.rows,
          (float)out_scale, (int)a.is_2d, (int)b.is_2d, dtype_code(c.scalar_type()), (int)a.packed};
}
bool product(Failure& f, const Copy& a, const Tensor& a_buf, const Copy& b, const Tensor& b_buf, const Tensor& c, double out_scale, void* s) {
  const alto_mxfp4_product p = product_of(a, a_buf, b, b_buf, c, out_scale);
  if (p.packed)
    return f.ok("alto_mxfp4_gemm_ps", api.gemm_ps(p.a, p.lda, p.a_scales, p.b, p.ldb, p.b_scales, p.M, p.N, p.K, p.c, p.ldc, p.out_scale, s));
  return f.ok("alto_mxfp4_gemm", api.gemm(p.a, p.lda, p.a_scales, p.a_ss_r, p.a_ss_k, p.a_is_2d, p.b, p.ldb, p.b_scales, p.b_ss_r, p.b_ss_k, p.b_is_2d, p.M, p.N, p.K, p.c,
                                          p.c_dtype, p.ldc, p.out_scale, s));
}

// linear.py:packed_gemm_supported
bool packed_gemm_supported(int64_t M, int64_t N, int64_t K) {
  return M >= 128 && N >= 128 && K >= 512 && N % 8 == 0 && M * (K / 2) < (1ll << 31) && N * (K / 2) < (1ll << 31);
}

// What a linear layer's step quantizes: x [M, K] (row, col), W [N, K] (row, col), dY [M, N] (row, col)
struct LinearCopies {
  Copy x_row, w_row, x_col, w_col, go_row, go_col;
  // packed: bits 0, 1, 2 = scales of the forward's, the input gradient's and the weight gradient's operands
  LinearCopies(int64_t M, int64_t N, int64_t K, int packed) {
    const bool f = packed & 1, d = packed & 2, w = packed & 4;
    x_row = {M, K, 1, 0, f, false};
    w_row = {N, K, 1, x_row.end(), f, !f};
    x_col = {K, M, 1, 0, w, false};
    w_col = {K, N, 1, 0, d, !d};
    go_row = {M, N, 1, 0, d, false};
    go_col = {N, M, 1, go_row.end(), w, false};
  }
};

void* current_stream(const Tensor& t) { return c10::hip::getCurrentHIPStream(t.device().index()).stream(); }

// A refused launch on its way out of a node
struct Refused {
  Failure failure;
};

// Inside the engine an error of the interpreter travels as torch's own exception
template <typename F>
auto with_interpreter(F&& f) {
  const py::gil_scoped_acquire gil;
  try {
    return f();
  } catch (py::error_already_set& e) {
    e.restore();
    python_error error;
    error.persist();
    throw error;
  }
}
void raise_in_engine(const Failure& f) {
  if (f.rc != 0) with_interpreter([&] { f.raise(); });
}
// (a module that is loaded: a lookup)
py::object python_function(const char* module, const char* name) { return py::module_::import(module).attr(name); }
// Forward-mode tangents of what comes into a node's backward would be lost there
void refuse_tangents(const char* what, const std::vector<Tensor>& grads) {
  for (const Tensor& g : grads)
    if (g.defined() && g._fw_grad(0).defined()) with_interpreter([&] { python_function("alto_amd.mxfp4._runtime", "refuse_transforms")(what, g); });
}
bool host_keyed_hardware_rounding() {
  return with_interpreter([] { return python_function("alto_amd.mxfp4._runtime", "host_keyed_hardware_rounding")().cast<bool>(); });
}

using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

std::string to_text(const StepOptions& o) { return std::string(reinterpret_cast<const char*>(&o), sizeof o); }
StepOptions options_of(AutogradContext* ctx) {
  StepOptions o;
  const std::string& text = ctx->saved_data["options"].toStringRef();
  std::memcpy(&o, text.data(), sizeof o);
  return o;
}
static_assert(std::is_trivially_copyable<StepOptions>::value, "kept as bytes");
py::object signs_of(const StepOptions& o) { return o.hadamard ? py::cast(at::from_blob(const_cast<int8_t*>(o.signs), {32}, at::kChar).clone()) : py::none(); }
py::object perm_of(const StepOptions& o) { return o.permuted ? py::cast(at::from_blob(const_cast<uint8_t*>(o.perm), {32}, at::kByte).clone()) : py::none(); }

struct StepOperands {   // what a node's forward works on, beside the tensors that its gradients belong to
  Tensor x, w, offs;    // x [M, K]; the plain weight behind a wrapper; groups (offsets or ends)
  bool ends = false;
  StepOptions o;
};
bool whole_buffer(const Tensor& t, int64_t n) { return on_gpu(t) && t.scalar_type() == at::kByte && t.dim() == 1 && t.numel() == n && t.is_contiguous() && aligned16(t); }

// philox_seed_offset(None, None)[0] of _runtime.py: the same draw
uint64_t draw_seed() { return (uint64_t)at::randint(0, INT64_MAX, {1}, at::TensorOptions().dtype(at::kLong).device(at::kCPU)).item<int64_t>(); }

// -> (dx, dw), or false; sr: the hardware's stochastic converts, keyed with a draw from torch's CPU generator
bool linear_gradients(const Tensor& go_in, const Tensor& xs, const Tensor& ws, const StepOptions& o, Tensor& dx, Tensor& dw) {
  const int64_t N = o.N, K = o.K;
  if (!on_gpu(go_in) || go_in.scalar_type() != o.dtype || go_in.dim() < 2 || go_in.size(-1) != N) return false;
  const Tensor go = go_in.dim() == 2 ? go_in : go_in.reshape({-1, N});
  const int64_t M = go.size(0);
  const LinearCopies c(M, N, K, o.packed);
  if (!rows_readable(go) || !whole_buffer(xs, c.x_col.end()) || !whole_buffer(ws, c.w_col.end())) return false;
  if (o.packed != 0 && go.scalar_type() != at::kBFloat16) return false;
  if (o.sr && !host_keyed_hardware_rounding()) return false;
  const Hadamard h(o);
  Failure f;
  const uint64_t seed = o.sr ? draw_seed() : 0;
  const Tensor tmp = Alloc(go).dense({c.go_col.end()});
  dx = at::empty({M, K}, go.options());
  dw = at::empty({N, K}, go.options());
  void* s = current_stream(go);
  quantize_gradient(f, go, c.go_row, tmp, c.go_col, tmp, o.sr ? 3 : 0, seed, h, o.clip, o.uos, s) && [&] {
    const alto_mxfp4_product x = product_of(c.go_row, tmp, c.w_col, ws, dx, 1.0), w = product_of(c.go_col, tmp, c.x_col, xs, dw, o.out_scale);
    return f.ok("alto_mxfp4_gemm_two", api.gemm_two(&x, &w, s));
  }();
  raise_in_engine(f);
  if (go_in.dim() != 2) {
    auto shape = go_in.sizes().vec();
    shape.back() = K;
    dx = dx.view(shape);
  }
  return true;
}

struct LinearNode : torch::autograd::Function<LinearNode> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x_in, const Tensor&, const StepOperands& op) {
    const StepOptions& o = op.o;
    const int64_t M = op.x.size(0);
    const LinearCopies c(M, o.N, o.K, o.packed);
    const Hadamard h(o);
    Failure f;
    const Alloc a(op.x);
    const Tensor tmp = a.dense({c.w_row.end()}), xs = a.dense({c.x_col.end()}), ws = a.dense({c.w_col.end()});
    const Tensor y = at::empty({M, o.N}, op.x.options());
    void* s = current_stream(op.x);
    quantize_operands(f, op.x, c.x_row, tmp, c.x_col, xs, h, o.clip, op.w, c.w_row, tmp, c.w_col, ws, o.uos, s) && product(f, c.x_row, tmp, c.w_row, tmp, y, 1.0, s);
    if (f.rc != 0) throw Refused{f};
    ctx->save_for_backward({xs, ws});
    ctx->saved_data["options"] = to_text(o);
    // a view for two dimensions as well, as the general function returns it: autograd refuses to change either in place
    auto shape = x_in.sizes().vec();
    shape.back() = o.N;
    return y.view(shape);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const StepOptions o = options_of(ctx);
    const variable_list saved = ctx->get_saved_variables();
    variable_list out(3);   // x, the weight, the operands
    if (!linear_gradients(grads[0], saved[0], saved[1], o, out[0], out[1]))
      with_interpreter([&] {
        const py::tuple g = python_function("alto_amd.mxfp4.linear", "_declined_backward")(grads[0], saved[0], saved[1], o.N, o.K, o.packed, o.dtype == at::kBFloat16, o.sr,
                                                                                          signs_of(o), perm_of(o), o.clip, o.uos, o.dge);
        out[0] = g[0].cast<Tensor>();
        out[1] = g[1].cast<Tensor>();
      });
    return out;
  }
};

template <typename Node>
py::object apply_node(const Tensor& x, const Tensor& weight, const StepOperands& op) {
  Tensor y;
  Failure f;
  {
    py::gil_scoped_release nogil;
    try {
      y = Node::apply(x, weight, op);
    } catch (const Refused& r) {
      f = r.failure;
    }
  }
  f.raise();
  return py::cast(y);
}

// linear.py:MXFP4LinearStep -> y, or None.  `weight`: what the gradient belongs to (a wrapper, perhaps), `w`: its values
py::object linear_step(const Tensor& x, const Tensor& weight, const Tensor& w, const OptTensor& signs, const OptTensor& perm, int clip, bool uos, bool sr, bool dge,
                       double out_scale, bool allow_packed) {
  if (!on_gpu(x) || x.dim() < 2 || w.dim() != 2 || !rows_readable(w) || !node_serves(x, weight)) return py::none();
  StepOperands op{x, w, Tensor(), false, StepOptions(signs, perm, clip, uos, sr, dge, out_scale)};
  const int64_t N = op.o.N = w.size(0), K = op.o.K = w.size(1);
  if (x.size(-1) != K || x.numel() == 0 || N == 0 || N % 32 != 0 || K % 32 != 0) return py::none();
  if (x.dim() != 2) {
    const at::NoGradGuard guard;
    op.x = x.reshape({-1, K});
  }
  const int64_t M = op.x.size(0);
  if (M % 32 != 0 || !rows_readable(op.x)) return py::none();
  op.o.dtype = x.scalar_type();
  if (allow_packed && op.o.dtype == at::kBFloat16 && M * std::max(N, K) < (1ll << 36) && N * K < (1ll << 36))
    op.o.packed = (int)packed_gemm_supported(M, N, K) | (int)packed_gemm_supported(M, K, N) << 1 | (int)packed_gemm_supported(N, K, M) << 2;
  return apply_node<LinearNode>(x, weight, op);
}

// (a saved-tensor hook may hand a buffer back at any address)
Tensor whole_aligned(const Tensor& t) { return t.is_contiguous() && aligned16(t) ? t : t.clone(at::MemoryFormat::Contiguous); }

// The saved buffers as the four tensors that MXFP4LinearFunction saves: column codes and scales of x and of W
py::tuple linear_saved(const Tensor& xs_in, const Tensor& ws_in, int64_t M, int64_t N, int64_t K, int packed) {
  const LinearCopies c(M, N, K, packed);
  const Tensor xs = whole_aligned(xs_in), ws = whole_aligned(ws_in);
  auto codes = [](const Tensor& b, const Copy& k) { return b.as_strided({k.K / 2, k.rows}, {1, k.ld()}, b.storage_offset() + k.at); };
  auto scales = [](const Tensor& b, const Copy& k) {
    const int64_t o = b.storage_offset() + k.scales_at();
    if (k.packed) return b.as_strided({div_up(k.K / 32, 16), k.rows, 16}, {k.rows * 16, 16, 1}, o);
    return b.as_strided({k.K / 32, k.is_2d ? k.rows / 32 : k.rows}, {1, k.scale_ld()}, o);
  };
  return py::make_tuple(codes(xs, c.x_col), scales(xs, c.x_col), codes(ws, c.w_col), scales(ws, c.w_col));
}

// grouped_gemm.py:grouped_packed_supported and grouped_dw_packed_supported
bool grouped_packed_supported(int64_t M, int64_t N, int64_t K, int64_t groups) {
  const int64_t ld = div_up(K / 2, 16) * 16;
  return M >= 128 && N >= 128 && K >= 512 && N % 8 == 0 && M * ld < (1ll << 31) && N * ld < (1ll << 31) && div_up(K / 32, 16) * std::max(M, N) * 16 < (1ll << 31) &&
         (div_up(M, 256) + groups + 2) * div_up(N, 256) < (1ll << 28);
}
bool grouped_dw_packed_supported(int64_t M, int64_t N, int64_t K, int64_t groups, int64_t experts) {
  const int64_t ld = div_up(M / 2, 16) * 16;
  return M >= 512 && M % 32 == 0 && N >= 128 && K >= 128 && N % 8 == 0 && K % 8 == 0 && N * ld < (1ll << 31) && K * ld < (1ll << 31) && groups <= 32768 && experts <= 65535 &&
         div_up(M, 512) * std::max(N, K) * 16 < (1ll << 31);
}

// What a grouped layer's step quantizes, all scales packed: x [M, K], dY [M, N] as above; the experts in one pass over their storage
// ([E, N, K], or [E, K, N]): copies packed along K for the forward and along N for the input gradient
struct GroupedCopies {
  Copy x_row, x_col, wf, wd, go_row, go_col;
  GroupedCopies(int64_t M, int64_t E, int64_t N, int64_t K) {
    x_row = {M, K, 1, 0, true, false};
    wf = {N, K, E, x_row.end(), true, true};
    x_col = {K, M, 1, 0, true, false};
    wd = {K, N, E, 0, true, true};
    go_row = {M, N, 1, 0, true, false};
    go_col = {N, M, 1, go_row.end(), true, false};
  }
};

bool grouped_product(Failure& f, const Copy& a, const Tensor& a_buf, const Copy& w, const Tensor& w_buf, const Tensor& offs, const Tensor& plan, bool planned,
                     const Tensor& out, void* s) {
  return f.ok("alto_mxfp4_grouped_gemm_ps",
              api.grouped_gemm_ps(a.codes(a_buf), a.ld(), a.scales(a_buf), w.codes(w_buf), w.rows * w.ld(), w.ld(), w.scales(w_buf), w.scale_bytes(),
                                  static_cast<const int32_t*>(offs.data_ptr()), nullptr, (int)w.batch, (int)w.batch, a.rows, w.rows, a.K, out.data_ptr(), w.rows,
                                  plan.data_ptr(), plan.numel(), (int)planned, s));
}

// -> (dx, dw), or false
bool grouped_gradients(const Tensor& go, const Tensor& xs, const Tensor& ws, const Tensor& offs, const Tensor& plan, const StepOptions& o, Tensor& dx, Tensor& dw) {
  const int64_t E = o.E, N = o.N, K = o.K;
  if (go.dim() != 2 || go.size(1) != N || !rows_readable(go) || go.scalar_type() != at::kBFloat16 || !go.is_contiguous()) return false;
  const int64_t M = go.size(0);
  const GroupedCopies c(M, E, N, K);
  if (!whole_buffer(xs, c.x_col.end()) || !whole_buffer(ws, c.wd.end()) || !whole_buffer(plan, api.grouped_gemm_workspace_bytes(M, (int)E))) return false;
  if (!on_gpu(offs) || offs.scalar_type() != at::kInt || offs.numel() != E + 1 || !offs.is_contiguous()) return false;
  if (o.sr && !host_keyed_hardware_rounding()) return false;
  const Hadamard h(o);
  Failure f;
  const uint64_t seed = o.sr ? draw_seed() : 0;
  void* s = current_stream(go);
  const Tensor tmp = Alloc(go).dense({c.go_col.end()});
  dx = at::empty({M, K}, go.options());
  dw = o.trans_weights ? at::empty({E, N, K}, go.options()) : at::empty({E, K, N}, go.options());
  const Copy &g = c.go_row, &w = c.wd, &gt = c.go_col, &xt = c.x_col;
  quantize_gradient(f, go, g, tmp, gt, tmp, o.sr ? 3 : 0, seed, h, o.clip, o.uos, s) &&
      f.ok("alto_mxfp4_grouped_gradients_ps",
           api.grouped_gradients_ps(g.codes(tmp), g.ld(), g.scales(tmp), w.codes(ws), w.rows * w.ld(), w.ld(), w.scales(ws), w.scale_bytes(), gt.codes(tmp), gt.ld(),
                                    gt.scales(tmp), xt.codes(xs), xt.ld(), xt.scales(xs), static_cast<const int32_t*>(offs.data_ptr()), (int)E, M, N, K, dx.data_ptr(), K,
                                    dw.data_ptr(), dw.stride(0), o.trans_weights ? dw.stride(1) : dw.stride(2), o.trans_weights ? dw.stride(2) : dw.stride(1),
                                    (float)o.out_scale, plan.data_ptr(), plan.numel(), s));
  raise_in_engine(f);
  return true;
}

struct GroupedNode : torch::autograd::Function<GroupedNode> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor&, const StepOperands& op) {
    const StepOptions& o = op.o;
    const int64_t M = x.size(0), E = o.E;
    const GroupedCopies c(M, E, o.N, o.K);
    const Hadamard h(o);
    Failure f;
    const Alloc a(op.x);
    void* s = current_stream(op.x);
    const Tensor tmp = a.dense({c.wf.end()}), xs = a.dense({c.x_col.end()}), ws = a.dense({c.wd.end()});
    const Tensor out = at::empty({M, o.N}, op.x.options()), plan = a.dense({api.grouped_gemm_workspace_bytes(M, (int)E)});
    Tensor offs = op.offs;
    bool ok = true;
    if (op.ends) {
      offs = at::empty({E + 1}, op.offs.options());
      ok = f.ok("alto_mxfp4_grouped_gemm_plan_ends", api.grouped_gemm_plan_ends(static_cast<const int32_t*>(op.offs.data_ptr()), (int)E, static_cast<int32_t*>(offs.data_ptr()), M,
                                                                                plan.data_ptr(), plan.numel(), s));
    }
    ok = ok && (o.trans_weights ? quantize_operands(f, op.x, c.x_row, tmp, c.x_col, xs, h, o.clip, op.w, c.wf, tmp, c.wd, ws, o.uos, s)
                                : quantize_operands(f, op.x, c.x_row, tmp, c.x_col, xs, h, o.clip, op.w, c.wd, ws, c.wf, tmp, o.uos, s));
    ok = ok && grouped_product(f, c.x_row, tmp, c.wf, tmp, offs, plan, op.ends, out, s);
    if (!ok) throw Refused{f};
    ctx->save_for_backward({xs, ws, offs, plan});
    ctx->saved_data["options"] = to_text(o);
    return out;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const StepOptions o = options_of(ctx);
    const variable_list saved = ctx->get_saved_variables();
    variable_list out(3);   // x, the weights, the operands
    if (!grouped_gradients(grads[0], saved[0], saved[1], saved[2], saved[3], o, out[0], out[1]))
      with_interpreter([&] {
        const py::tuple g = python_function("alto_amd.mxfp4.grouped_gemm", "_declined_backward")(grads[0], saved[0], saved[1], saved[2], saved[3], o.E, o.N, o.K, o.trans_weights,
                                                                                                o.sr, signs_of(o), perm_of(o), o.clip, o.uos, o.dge);
        out[0] = g[0].cast<Tensor>();
        out[1] = g[1].cast<Tensor>();
      });
    return out;
  }
};

// grouped_gemm.py:MXFP4GroupedStep: x [M, K] bf16, w [E, N, K] (trans) or [E, K, N], groups as offsets [E + 1] or, with `ends`, as
// cumulative group ends [E] -> out, or None
py::object grouped_step(const Tensor& x, const Tensor& weight, const Tensor& w, const Tensor& offs, bool ends, bool trans_weights, const OptTensor& signs, const OptTensor& perm,
                        int clip, bool uos, bool sr, bool dge, double out_scale) {
  if (x.dim() != 2 || w.dim() != 3 || !rows_readable(x) || !rows_readable(w) || x.scalar_type() != at::kBFloat16 || !x.is_contiguous() || !w.is_contiguous()) return py::none();
  if (!node_serves(x, weight) || !on_gpu(offs) || offs.dim() != 1 || offs.scalar_type() != at::kInt || !offs.is_contiguous()) return py::none();
  const int64_t M = x.size(0), E = w.size(0), N = w.size(trans_weights ? 1 : 2), K = w.size(trans_weights ? 2 : 1);
  if (x.size(1) != K || offs.numel() != E + !ends || M == 0 || E == 0 || N % 32 != 0 || K % 32 != 0) return py::none();
  if (M * std::max(N, K) >= (1ll << 36) || N * K >= (1ll << 36) || !grouped_packed_supported(M, N, K, E) || !grouped_packed_supported(M, K, N, E) ||
      !grouped_dw_packed_supported(M, N, K, E, E))
    return py::none();
  StepOperands op{x, w, offs, ends, StepOptions(signs, perm, clip, uos, sr, dge, out_scale)};
  op.o.E = E; op.o.N = N; op.o.K = K;
  op.o.trans_weights = trans_weights;
  op.o.dtype = at::kBFloat16;
  return apply_node<GroupedNode>(x, weight, op);
}

// The saved buffers as the four tensors that MXFP4GroupedGEMM saves: token-packed codes and scales of x, codes [E, K, N / 2] and scales of W
py::tuple grouped_saved(const Tensor& xs_in, const Tensor& ws_in, int64_t M, int64_t E, int64_t N, int64_t K) {
  const GroupedCopies c(M, E, N, K);
  const Tensor xs = whole_aligned(xs_in), ws = whole_aligned(ws_in);
  const Copy &x = c.x_col, &w = c.wd;
  const int64_t xo = xs.storage_offset(), wo = ws.storage_offset();
  return py::make_tuple(xs.as_strided({M / 2, K}, {1, x.ld()}, xo + x.at), xs.as_strided({div_up(M / 32, 16), K, 16}, {K * 16, 16, 1}, xo + x.scales_at()),
                        ws.as_strided({E, K, N / 2}, {K * w.ld(), w.ld(), 1}, wo + w.at),
                        ws.as_strided({E, div_up(N / 32, 16), K, 16}, {w.scale_bytes(), K * 16, 16, 1}, wo + w.scales_at()));
}

// hadamard.py:HadamardFactory.create_transform: the same two draws (randint in the factory's dtype, then randperm) as int8
// signs and uint8 positions
py::tuple draw_hadamard(const std::optional<at::Generator>& gen, at::ScalarType dtype) {
  const auto cpu = at::TensorOptions().device(at::kCPU);
  Tensor q = at::randint(0, 2, {32}, gen, cpu.dtype(dtype));
  const Tensor p = at::randperm(32, gen, cpu.dtype(at::kLong));
  if (dtype != at::kFloat) q = q.to(at::kFloat);   // (zeros and ones)
  const Tensor signs = at::empty({32}, cpu.dtype(at::kChar)), perm = at::empty({32}, cpu.dtype(at::kByte));
  const float* qv = q.data_ptr<float>();
  const int64_t* pv = p.data_ptr<int64_t>();
  int8_t* sv = signs.data_ptr<int8_t>();
  uint8_t* mv = perm.data_ptr<uint8_t>();
  for (int i = 0; i < 32; ++i) {
    sv[i] = qv[i] != 0.0f ? 1 : -1;
    mv[i] = (uint8_t)pv[i];
  }
  return py::make_tuple(signs, perm);
}

// -------------------------------------------------------------------------------------------------- attention and its gradients
// What the backward takes beside the gradient of the output: quantized operands, the forward's results, the additive terms as _additive gives them
struct AttentionKept {
  Tensor q, q_scale, k, k_scale, v, v_scale, out, lse;
  OptTensor bias, slopes;
  double sm_scale = 0;
  bool causal = false, rows_outer = false;
  int64_t keys = 0;
  std::vector<int32_t> cu_q, cu_k;
};

// attention.py:_gradients -> {dq, dk, dv} (undefined: not wanted), or false: declined
bool attention_gradients(Failure& f, const Tensor& go_in, const AttentionKept& x, bool want_q, bool want_kv, variable_list& grads) {
  const Tensor &q = x.q, &k = x.k, &v = x.v;
  if (!node_serves(go_in, x.out) || x.lse._fw_grad(0).defined()) return false;
  for (const OptTensor* t : {&x.bias, &x.slopes})
    if (t->has_value() && (*t)->_fw_grad(0).defined()) return false;
  for (const Tensor* t : {&q, &x.q_scale, &k, &x.k_scale, &v, &x.v_scale})
    if (!on_current_device(*t) || t->scalar_type() != at::kByte || t->dim() != 4 || !t->is_contiguous()) return false;
  for (const Tensor* t : {&go_in, &x.out})
    if (!on_current_device(*t) || t->scalar_type() != at::kBFloat16 || t->dim() != 4) return false;
  const int64_t B = q.size(0), Hq = q.size(1), Sq = q.size(2), D = 2 * q.size(3), Hk = k.size(1), Sk = k.size(2), Dv = v.size(2);
  auto is = [](const Tensor& t, at::IntArrayRef size) { return t.sizes() == size; };
  if (!is(k, {B, Hk, Sk, D / 2}) || !is(v, {B, Hk, Dv, Sk / 2}) || !is(x.q_scale, {B, Hq, Sq / 32, D / 32}) || !is(x.k_scale, {B, Hk, Sk / 32, D / 32}) ||
      !is(x.v_scale, {B, Hk, Sk / 32, Dv / 32}) || !is(go_in, {B, Hq, Sq, Dv}) || !is(x.out, {B, Hq, Sq, Dv}))
    return false;
  if (!on_current_device(x.lse) || x.lse.scalar_type() != at::kFloat || !is(x.lse, {B, Hq, Sq}) || x.cu_q.size() != x.cu_k.size() || x.cu_q.size() == 1) return false;
  for (const OptTensor* t : {&x.bias, &x.slopes})
    if (t->has_value() && (!on_current_device(**t) || (*t)->scalar_type() != at::kFloat)) return false;
  const Tensor go = readable_rows(go_in), out = readable_rows(x.out);
  const auto opts = at::TensorOptions().dtype(at::kBFloat16).device(q.device());
  auto grad = [&](bool want, int64_t H, int64_t S, int64_t n) {
    if (!want) return Tensor();
    return x.rows_outer ? at::empty({B, S, H, n}, opts).transpose(1, 2) : at::empty({B, H, S, n}, opts);
  };
  const Tensor dq = grad(want_q, Hq, Sq, D), dk = grad(want_kv, Hk, Sk, D), dv = grad(want_kv, Hk, Sk, Dv);
  alto_mxfp4_attention_bwd_t a{};
  a.q_codes = bytes(q); a.q_scales = bytes(x.q_scale); a.k_codes = bytes(k); a.k_scales = bytes(x.k_scale); a.vt_codes = bytes(v); a.v_scales = bytes(x.v_scale);
  a.dout = bytes(go); a.out = bytes(out); a.lse = static_cast<const float*>(x.lse.data_ptr());
  a.dq = bytes(dq); a.dk = bytes(dk); a.dv = bytes(dv);
  a.B = B; a.Hq = Hq; a.Hk = Hk; a.Sq = Sq; a.Sk = Sk; a.Sk_used = x.keys; a.D = D; a.Dv = Dv;
  auto strides = [](const Tensor& t, int64_t& sb, int64_t& sh, int64_t& ss) {
    if (!t.defined()) return;
    sb = stride_of(t, 0); sh = stride_of(t, 1); ss = stride_of(t, 2);
  };
  strides(go, a.dout_sb, a.dout_sh, a.dout_ss);
  strides(out, a.out_sb, a.out_sh, a.out_ss);
  strides(x.lse, a.lse_sb, a.lse_sh, a.lse_ss);
  strides(dq, a.dq_sb, a.dq_sh, a.dq_ss);
  strides(dk, a.dk_sb, a.dk_sh, a.dk_ss);
  strides(dv, a.dv_sb, a.dv_sh, a.dv_ss);
  if (x.bias.has_value()) {
    a.bias = static_cast<const float*>(x.bias->data_ptr());
    a.bias_sb = stride_of(*x.bias, 0); a.bias_sh = stride_of(*x.bias, 1); a.bias_sm = x.bias->stride(2);
  }
  if (x.slopes.has_value()) {
    a.alibi_slopes = static_cast<const float*>(x.slopes->data_ptr());
    a.alibi_sb = stride_of(*x.slopes, 0); a.alibi_sh = x.slopes->stride(1);
  }
  if (!x.cu_q.empty()) { a.cu_q = x.cu_q.data(); a.cu_k = x.cu_k.data(); a.n_seqs = (int)x.cu_q.size() - 1; }
  a.causal = x.causal; a.sm_scale = (float)x.sm_scale;
  a.workspace_bytes = api.attention_bwd_workspace_bytes(&a);
  if (a.workspace_bytes < 0) return false;   // (the general path words the error)
  const Tensor ws = Alloc(q).dense({a.workspace_bytes});
  a.workspace = ws.data_ptr();
  f.ok("alto_mxfp4_attention_bwd", api.attention_bwd(&a, current_stream(q)));
  grads = {dq, dk, dv};
  return true;
}
py::object opt(const Tensor& t) { return t.defined() ? py::cast(t) : py::none(); }
py::object attention_gradients_py(const Tensor& go, const Tensor& q, const Tensor& q_scale, const Tensor& k, const Tensor& k_scale, const Tensor& v, const Tensor& v_scale,
                                  const Tensor& out, const Tensor& lse, double sm_scale, bool causal, int64_t seqlen_k, const OptTensor& bias, const OptTensor& slopes,
                                  const std::vector<int32_t>& cu_q, const std::vector<int32_t>& cu_k, bool rows_outer, bool want_q, bool want_kv) {
  Failure f;
  variable_list grads;
  {
    py::gil_scoped_release nogil;
    if (!attention_gradients(f, go, {q, q_scale, k, k_scale, v, v_scale, out, lse, bias, slopes, sm_scale, causal, rows_outer, seqlen_k, cu_q, cu_k}, want_q, want_kv, grads))
      grads.clear();
  }
  f.raise();
  return grads.empty() ? py::none() : py::object(py::make_tuple(opt(grads[0]), opt(grads[1]), opt(grads[2])));
}

// attention.py:MXFP4AttentionFunction without additive terms, as one native call a direction: as a Python function a forward of small sizes with a graph
// took 44 us, here 18 (without one 16).  Q is quantized ahead of the attention kernel, because the backward needs its codes, and not in it: 2048 tokens of
// 32 / 8 heads of 128 take 43 us for 40, 4 x 2048 of 64 / 8 185 for 173, 8192 of 16 / 2 145.5 for 146.3.
struct AttentionShape {
  int64_t B, Hq, Hk, Sq, Sk, D, Dv;
  double sm_scale;
  bool causal, rows_outer;
  // of the kept buffer: codes and scales of Q, K and V, 16 bytes of room behind each (the attention kernel reads scale bytes in whole dwords)
  int64_t bytes_of(int i) const {
    const int64_t n[6] = {B * Hq * Sq * D / 2, B * Hq * (Sq / 32) * (D / 32), B * Hk * Sk * D / 2, B * Hk * (Sk / 32) * (D / 32), B * Hk * Sk * Dv / 2, B * Hk * (Sk / 32) * (Dv / 32)};
    return n[i];
  }
  int64_t start(int i) const {
    int64_t at = 0;
    for (int j = 0; j < i; ++j) at += div_up(bytes_of(j) + 16, 256) * 256;
    return at;
  }
};
static_assert(std::is_trivially_copyable<AttentionShape>::value, "kept as bytes");
template <typename T>
std::string bytes_text(const T* p, size_t n) { return std::string(reinterpret_cast<const char*>(p), n * sizeof(T)); }

struct AttentionOperands {
  AttentionShape shape;
  bool lse_rows_outer;
  std::vector<int32_t> cu_q, cu_k;
};

struct AttentionNode : torch::autograd::Function<AttentionNode> {
  static variable_list forward(AutogradContext* ctx, const Tensor& q_in, const Tensor& k_in, const Tensor& v_in, const AttentionOperands& op) {
    const AttentionShape& x = op.shape;
    const Tensor q = readable_rows(q_in), k = readable_rows(k_in), v = readable_rows(v_in);
    const int64_t out_rows = x.rows_outer ? x.Hq * x.Dv : x.Dv, out_heads = x.rows_outer ? x.Dv : x.Sq * x.Dv;
    const Tensor buf = Alloc(q).dense({x.start(6)});
    const Tensor out = at::empty_strided({x.B, x.Hq, x.Sq, x.Dv}, {x.Hq * x.Sq * x.Dv, out_heads, out_rows, 1}, buf.options().dtype(at::kBFloat16));
    const Tensor lse = at::empty_strided({x.B, x.Hq, x.Sq}, {x.Hq * x.Sq, op.lse_rows_outer ? 1 : x.Sq, op.lse_rows_outer ? x.Hq : 1}, buf.options().dtype(at::kFloat));
    uint8_t* p[6];
    for (int i = 0; i < 6; ++i) p[i] = bytes(buf) + x.start(i);
    void* s = current_stream(q);
    const int n = op.cu_q.empty() ? 0 : (int)op.cu_q.size() - 1;
    Failure f;
    f.ok("alto_mxfp4_attention_quantize",
         api.attention_quantize(q.data_ptr(), k.data_ptr(), v.data_ptr(), dtype_code(q.scalar_type()), x.B, x.Hq, x.Hk, x.Sq, x.Sk, x.D, x.Dv, stride_of(q, 0), stride_of(q, 1),
                                stride_of(q, 2), stride_of(k, 0), stride_of(k, 1), stride_of(k, 2), stride_of(v, 0), stride_of(v, 1), stride_of(v, 2), p[0], p[1], p[2], p[3],
                                p[4], p[5], s)) &&
        f.ok("alto_mxfp4_attention_fwd_strided",
             api.attention_fwd_strided(p[0], p[1], p[2], p[3], p[4], p[5], out.data_ptr(), static_cast<float*>(lse.data_ptr()), x.B, x.Hq, x.Hk, x.Sq, x.Sk, x.D, x.Dv,
                                       out.stride(0), out.stride(1), out.stride(2), lse.stride(0), lse.stride(1), lse.stride(2), n, n ? op.cu_q.data() : nullptr,
                                       n ? op.cu_k.data() : nullptr, (float)x.sm_scale, (int)x.causal, nullptr, 0, 0, s));
    if (f.rc != 0) throw Refused{f};
    ctx->save_for_backward({buf, out, lse});
    ctx->saved_data["shape"] = bytes_text(&x, 1);
    ctx->saved_data["cu_q"] = bytes_text(op.cu_q.data(), op.cu_q.size());
    ctx->saved_data["cu_k"] = bytes_text(op.cu_k.data(), op.cu_k.size());
    ctx->saved_data["dtype"] = (int64_t)q.scalar_type();
    ctx->mark_non_differentiable({lse});
    return {out, lse};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    refuse_tangents("attention", {grads[0]});
    const bool again = at::GradMode::is_enabled() && grads[0].requires_grad();
    const at::NoGradGuard guard;
    const variable_list saved = ctx->get_saved_variables();
    AttentionShape x;
    std::memcpy(&x, ctx->saved_data["shape"].toStringRef().data(), sizeof x);
    auto boundaries = [&](const char* name) {
      const std::string& text = ctx->saved_data[name].toStringRef();
      std::vector<int32_t> c(text.size() / sizeof(int32_t));
      if (!c.empty()) std::memcpy(c.data(), text.data(), text.size());
      return c;
    };
    const Tensor buf = whole_aligned(saved[0]);
    auto part = [&](int i, at::IntArrayRef size) { return buf.narrow(0, x.start(i), x.bytes_of(i)).view(size); };
    const AttentionKept kept{part(0, {x.B, x.Hq, x.Sq, x.D / 2}),       part(1, {x.B, x.Hq, x.Sq / 32, x.D / 32}), part(2, {x.B, x.Hk, x.Sk, x.D / 2}),
                             part(3, {x.B, x.Hk, x.Sk / 32, x.D / 32}), part(4, {x.B, x.Hk, x.Dv, x.Sk / 2}),      part(5, {x.B, x.Hk, x.Sk / 32, x.Dv / 32}),
                             saved[1], saved[2], std::nullopt, std::nullopt, x.sm_scale, x.causal, x.rows_outer, x.Sk, boundaries("cu_q"), boundaries("cu_k")};
    const bool need[3] = {ctx->needs_input_grad(0), ctx->needs_input_grad(1), ctx->needs_input_grad(2)};
    variable_list out;
    Failure f;
    if (!attention_gradients(f, grads[0], kept, need[0], need[1] || need[2], out))
      with_interpreter([&] {   // (what the native form declines: the general form serves it, or words the error)
        const py::tuple operands = py::make_tuple(kept.q, kept.q_scale, kept.k, kept.k_scale, kept.v, kept.v_scale);
        const py::tuple g = python_function("alto_amd.mxfp4.attention", "_gradients")(grads[0], operands, kept.out, kept.lse, kept.sm_scale, kept.causal, kept.keys, py::none(),
                                                                                     py::none(), kept.cu_q, kept.cu_k, kept.rows_outer, need[0], need[1] || need[2]);
        out.resize(3);
        for (int i = 0; i < 3; ++i)
          if (!g[i].is_none()) out[i] = g[i].cast<Tensor>();
      });
    raise_in_engine(f);
    const at::ScalarType dtype = (at::ScalarType)ctx->saved_data["dtype"].toInt();
    for (int i = 0; i < 3; ++i) {
      if (!need[i]) out[i] = Tensor();
      else if (out[i].scalar_type() != dtype) out[i] = out[i].to(dtype);
    }
    if (again) {   // (the gradients have none of their own: a second derivative ends in an error, as of a function marked once_differentiable)
      for (Tensor& g : out)
        if (g.defined()) g = g.detach().set_requires_grad(true);
      const at::AutoGradMode on(true);
      out = std::make_shared<torch::autograd::DelayedError>("the gradients of attention are not differentiable", 3)->apply(std::move(out));
    }
    out.emplace_back();   // (the operands)
    return out;
  }
};

// Attention of everyday calls whose Q, K or V require a gradient -> (out, lse) with their graph, or None
py::object attention_step(const Tensor& q, const Tensor& k, const Tensor& v, double sm_scale, bool causal, bool rows_outer, bool lse_rows_outer, const std::vector<int32_t>& cu_q,
                          const std::vector<int32_t>& cu_k) {
  for (const Tensor* t : {&q, &k, &v})
    if (!on_current_device(*t) || !is_float(*t) || t->dim() != 4 || t->scalar_type() != q.scalar_type() || t->numel() == 0) return py::none();
  if (!node_serves(q, k) || v._fw_grad(0).defined() || cu_q.size() != cu_k.size()) return py::none();
  const AttentionShape x{q.size(0), q.size(1), v.size(1), q.size(2), v.size(2), q.size(3), v.size(3), sm_scale, causal, rows_outer};
  if (k.size(0) != x.B || v.size(0) != x.B || k.size(1) != x.Hk || k.size(2) != x.Sk || k.size(3) != x.D) return py::none();
  if (x.Sq % 32 != 0 || x.Sk % 32 != 0 || x.D % 32 != 0 || x.Dv % 32 != 0) return py::none();
  variable_list out;
  Failure f;
  {
    py::gil_scoped_release nogil;
    try {
      out = AttentionNode::apply(q, k, v, AttentionOperands{x, lse_rows_outer, cu_q, cu_k});
    } catch (const Refused& r) {
      f = r.failure;
    }
  }
  f.raise();
  return py::make_tuple(out[0], out[1]);
}

// ------------------------------------------------------------------------------------------------------------ rotary positions
// rotary.py:apply_rotary and its backward.  As Python functions around one native call each a forward took 21 us and a training step 145
// (5.8 and 33 to 60 here: torch's engine and its thread).
struct RotaryOperands {
  Tensor inv_freq, positions;   // (positions undefined: 0, 1, ...)
  bool interleaved = false, inverse = false;
  double factor = 1.0;
  int64_t layout = 0;           // 0: [B, H, S, D], 1: [B, S, H, D], 2: [T, H, D]
  int64_t batch() const { return layout == 2 ? -1 : 0; }
  int64_t head() const { return layout == 0 ? 1 : layout == 1 ? 2 : 1; }
  int64_t row() const { return layout == 0 ? 2 : layout == 1 ? 1 : 0; }
};

// q and k rotated (either may be undefined: not wanted), of whatever strides
variable_list rotate(Failure& f, const Tensor& q_in, const Tensor& k_in, const RotaryOperands& op) {
  auto readable = [](const Tensor& t) { return !t.defined() || t.stride(-1) == 1 ? t : t.contiguous(); };
  Tensor q = readable(q_in), k = readable(k_in);
  if (!q.defined()) std::swap(q, k);
  variable_list out(2);
  Tensor q2 = at::empty(q.sizes(), q.options()), k2 = k.defined() ? at::empty(k.sizes(), k.options()) : Tensor();
  alto_mxfp4_rotary_t a{};
  a.q = q.data_ptr(); a.q_out = q2.data_ptr();
  if (k.defined()) { a.k = k.data_ptr(); a.k_out = k2.data_ptr(); a.Hk = k.size(op.head()); }
  a.inv_freq = static_cast<const double*>(op.inv_freq.data_ptr());
  a.B = op.batch() < 0 ? 1 : q.size(op.batch()); a.S = q.size(op.row()); a.Hq = q.size(op.head()); a.D = q.size(-1); a.R = 2 * op.inv_freq.size(0);
  auto strides = [&](const Tensor& t, int64_t& sb, int64_t& sh, int64_t& ss) {
    if (!t.defined()) return;
    sb = op.batch() < 0 ? 0 : stride_of(t, op.batch()); sh = stride_of(t, op.head()); ss = stride_of(t, op.row());
  };
  strides(q, a.q_sb, a.q_sh, a.q_ss);
  strides(k, a.k_sb, a.k_sh, a.k_ss);
  strides(q2, a.qo_sb, a.qo_sh, a.qo_ss);
  strides(k2, a.ko_sb, a.ko_sh, a.ko_ss);
  if (op.positions.defined()) {
    const Tensor& p = op.positions;
    a.positions = p.data_ptr();
    a.positions_are_32 = p.scalar_type() == at::kInt;
    a.pos_sb = p.dim() == 1 ? 0 : stride_of(p, 0); a.pos_ss = stride_of(p, p.dim() - 1);
  }
  a.factor = op.factor; a.dtype = dtype_code(q.scalar_type()); a.interleaved = op.interleaved; a.inverse = op.inverse;
  f.ok("alto_mxfp4_rotary", api.rotary(&a, current_stream(q)));
  out[q_in.defined() ? 0 : 1] = q2;
  if (k.defined()) out[1] = k2;
  return out;
}

struct RotaryNode : torch::autograd::Function<RotaryNode> {
  static variable_list forward(AutogradContext* ctx, const Tensor& q, const Tensor& k, const RotaryOperands& op) {
    Failure f;
    variable_list out = rotate(f, q, k, op);
    if (f.rc != 0) throw Refused{f};
    ctx->save_for_backward({op.inv_freq, op.positions});
    ctx->saved_data["interleaved"] = op.interleaved;
    ctx->saved_data["inverse"] = op.inverse;
    ctx->saved_data["factor"] = op.factor;
    ctx->saved_data["layout"] = op.layout;
    return out;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    refuse_tangents("apply_rotary", grads);
    const variable_list saved = ctx->get_saved_variables();
    RotaryOperands op;
    op.inv_freq = saved[0];
    op.positions = saved[1];
    op.interleaved = ctx->saved_data["interleaved"].toBool();
    op.inverse = !ctx->saved_data["inverse"].toBool();
    op.factor = ctx->saved_data["factor"].toDouble();
    op.layout = ctx->saved_data["layout"].toInt();
    variable_list out(3);   // q, k, the operands
    Failure f;
    if (at::GradMode::is_enabled() && (grads[0].requires_grad() || grads[1].requires_grad())) {   // (the rotation is linear: its gradient is one)
      try {
        const variable_list both = apply(grads[0], grads[1], op);
        out[0] = both[0];
        out[1] = both[1];
      } catch (const Refused& r) {
        f = r.failure;
      }
    } else {
      const variable_list both = rotate(f, ctx->needs_input_grad(0) ? grads[0] : Tensor(), ctx->needs_input_grad(1) ? grads[1] : Tensor(), op);
      out[0] = both[0];
      out[1] = both[1];
    }
    raise_in_engine(f);
    return out;
  }
};

// q and k of everyday calls -> (q, k) rotated, with their graph where they need one
py::object rotary(const Tensor& q, const Tensor& k, const Tensor& inv_freq, const OptTensor& positions, bool interleaved, double factor, int64_t layout) {
  const int64_t dims = layout == 2 ? 3 : 4;
  RotaryOperands op{inv_freq, positions.has_value() ? *positions : Tensor(), interleaved, false, factor, layout};
  for (const Tensor* t : {&q, &k})
    if (!on_current_device(*t) || !is_float(*t) || t->dim() != dims) return py::none();
  if (q.scalar_type() != k.scalar_type() || q.numel() == 0 || k.numel() == 0) return py::none();
  for (int64_t d = 0; d < dims; ++d)
    if (d != op.head() && q.size(d) != k.size(d)) return py::none();
  if (!on_current_device(inv_freq) || inv_freq.scalar_type() != at::kDouble || inv_freq.dim() != 1 || !inv_freq.is_contiguous() || inv_freq.requires_grad() || inv_freq._fw_grad(0).defined()) return py::none();
  if (inv_freq.size(0) < 1 || inv_freq.size(0) > 1024 || 2 * inv_freq.size(0) > q.size(-1)) return py::none();
  if (positions.has_value()) {
    const Tensor& p = *positions;
    if (!on_current_device(p) || (p.scalar_type() != at::kInt && p.scalar_type() != at::kLong)) return py::none();
    const int64_t S = q.size(op.row());
    if (!(p.dim() == 1 && p.size(0) == S) && !(layout != 2 && p.dim() == 2 && (p.size(0) == 1 || p.size(0) == q.size(0)) && p.size(1) == S)) return py::none();
  }
  if (!node_serves(q, k)) return py::none();
  variable_list out;
  Failure f;
  {
    py::gil_scoped_release nogil;
    if (at::GradMode::is_enabled() && (q.requires_grad() || k.requires_grad())) {
      try {
        out = RotaryNode::apply(q, k, op);
      } catch (const Refused& r) {
        f = r.failure;
      }
    } else {
      out = rotate(f, q, k, op);
    }
  }
  f.raise();
  return py::make_tuple(out[0], out[1]);
}

// ------------------------------------------------------------------------------------- 8-bit operands, a scale for each 128
// blockwise_fp8.py: the quantizer and the products.  (In Python a call took 16 us, most of it ahead of the launch.)
bool is_fp8(const Tensor& t) { return t.scalar_type() == at::kFloat8_e4m3fn || t.scalar_type() == at::kFloat8_e5m2; }
int fp8_code(at::ScalarType t) { return t == at::kFloat8_e4m3fn ? ALTO_FP8_E4M3 : ALTO_FP8_E5M2; }
bool is_offsets(const Tensor& t) { return on_current_device(t) && t.scalar_type() == at::kInt && t.dim() == 1 && t.size(0) >= 2 && t.is_contiguous(); }
// what neither wants a graph nor is being transformed
bool plain_operands(std::initializer_list<const Tensor*> all) {
  for (const Tensor* t : all)
    if (!on_current_device(*t) || t->is_neg() || (at::GradMode::is_enabled() && t->requires_grad()) || !node_serves(*t, *t)) return false;
  return true;
}

struct Fp8Copies {
  Tensor row, row_scales, col, col_scales;   // as quantize_blockwise_fp8_rowcol returns them
};
// x [M, C] or [B, M, C], neither empty, unit stride along C
Fp8Copies fp8_quantize_call(Failure& f, const Tensor& x, bool want_row, bool want_col, bool is_2d, at::ScalarType code, const Tensor& offs) {
  const bool batched = x.dim() == 3;
  const int64_t B = batched ? x.size(0) : 1, M = x.size(-2), C = x.size(-1), groups = offs.defined() ? offs.size(0) - 1 : 0;
  const int64_t tokens = offs.defined() ? 128 * api.fp8_token_blocks(M, groups) : M, mb = div_up(tokens, 128), cb = div_up(C, 128);
  const auto q = x.options().dtype(code).requires_grad(false), s = x.options().dtype(at::kFloat).requires_grad(false);
  auto make = [&](int64_t rows, int64_t cols, int64_t step_r, int64_t step_c, int64_t step_b) {
    return batched ? at::empty_strided({B, rows, cols}, {step_b, step_r, step_c}, s) : at::empty_strided({rows, cols}, {step_r, step_c}, s);
  };
  // codes of n rows at a pitch, the last one's pitch in their memory too (the quantizer writes, and products read, to the next multiple of 16 bytes)
  auto make_codes = [&](int64_t n, int64_t pitch, int64_t rows, int64_t cols, int64_t step_r, int64_t step_c) {
    const Tensor t = at::empty({B * n * pitch}, q);
    const int64_t size[] = {B, rows, cols}, step[] = {n * pitch, step_r, step_c};
    const int dims = batched ? 3 : 2;
    t.unsafeGetTensorImpl()->set_sizes_and_strides(at::IntArrayRef(size + 3 - dims, dims), at::IntArrayRef(step + 3 - dims, dims));
    return t;
  };
  Fp8Copies out;
  alto_mxfp4_fp8_quantize_t a{};
  if (is_2d) out.row_scales = out.col_scales = make(mb, cb, cb, 1, mb * cb);
  if (want_row) {
    const int64_t pitch = pitch128(C);
    out.row = make_codes(M, pitch, M, C, pitch, 1);
    if (!is_2d) out.row_scales = make(M, cb, 1, M, cb * M);
    a.row_codes = out.row.data_ptr(); a.row_ld = pitch; a.row_sb = M * pitch;
  }
  if (want_col) {
    const int64_t pitch = pitch128(tokens);
    out.col = make_codes(C, pitch, tokens, C, 1, pitch);
    if (!is_2d) out.col_scales = make(mb, C, C, 1, mb * C);
    a.col_codes = out.col.data_ptr(); a.col_ld = pitch; a.col_sb = C * pitch;
  }
  a.x = x.data_ptr();
  a.row_scales = out.row_scales.defined() ? static_cast<float*>(out.row_scales.data_ptr()) : nullptr;
  a.col_scales = out.col_scales.defined() ? static_cast<float*>(out.col_scales.data_ptr()) : nullptr;
  a.offs = offs.defined() ? static_cast<const int32_t*>(offs.data_ptr()) : nullptr;
  a.B = B; a.M = M; a.C = C; a.x_sb = batched ? stride_of(x, 0) : 0; a.x_sm = stride_of(x, x.dim() - 2);
  a.dtype = dtype_code(x.scalar_type()); a.code = fp8_code(code); a.is_2d = is_2d; a.groups = (int)groups;
  f.ok("alto_mxfp4_fp8_quantize", api.fp8_quantize(&a, current_stream(x)));
  return out;
}
py::object fp8_quantize(const Tensor& x, bool want_row, bool want_col, bool is_2d, bool e5m2, const OptTensor& offs) {
  if (!on_current_device(x) || !is_float(x) || x.dim() < 2 || x.dim() > 3 || x.numel() == 0 || x.is_neg() || !node_serves(x, x) || (x.size(-1) != 1 && x.stride(-1) != 1)) return py::none();
  if (offs.has_value() && (x.dim() != 2 || is_2d || !is_offsets(*offs))) return py::none();
  Failure f;
  Fp8Copies out;
  {
    py::gil_scoped_release nogil;
    out = fp8_quantize_call(f, x, want_row, want_col, is_2d, e5m2 ? at::kFloat8_e5m2 : at::kFloat8_e4m3fn, offs.has_value() ? *offs : Tensor());
  }
  f.raise();
  auto opt = [](const Tensor& t) -> py::object { return t.defined() ? py::cast(t) : py::none(); };
  return py::make_tuple(opt(out.row), opt(out.row_scales), opt(out.col), opt(out.col_scales));
}

// Codes as blockwise_fp8.py:_operand hands them on without a copy: dims of rows and of the reduction, the others in front
bool fp8_readable(const Tensor& t, int64_t row, int64_t k) {
  const int64_t rows = t.size(row), K = t.size(k), ld = stride_of(t, row);
  if ((K != 1 && t.stride(k) != 1) || ld % 16 != 0 || (rows > 1 && ld < K) || ld >= (1 << 22) || !aligned16(t)) return false;
  int64_t end = t.storage_offset() + (rows - 1) * ld + div_up(K, 16) * 16;
  if (t.dim() == 3) {
    if (stride_of(t, 0) % 16 != 0) return false;
    end += (t.size(0) - 1) * stride_of(t, 0);
  }
  return K % 16 == 0 || end <= (int64_t)t.storage().nbytes();
}
constexpr int64_t fp8_longest = (1 << 22) - 16;   // reduction of a native product; blockwise_fp8.py takes longer ones in parts
bool fp8_scales(const Tensor& s, int64_t row) { return s.scalar_type() == at::kFloat && stride_of(s, row) < (1 << 21); }
Tensor fp8_result(at::IntArrayRef size, const Tensor& like, at::ScalarType dtype) { return at::empty(size, at::TensorOptions().dtype(dtype).device(like.device())); }

// a [M, K] or, with trans_a, [K, M]; b [K, N] or, with trans_b, [N, K]; scales in the same orientation.  Undefined: declined
Tensor fp8_gemm_call(Failure& f, const Tensor& a, const Tensor& as, const Tensor& b, const Tensor& bs, bool a_2d, bool b_2d, bool trans_a, bool trans_b, at::ScalarType dtype) {
  if (a.dim() != 2 || b.dim() != 2 || as.dim() != 2 || bs.dim() != 2 || !is_fp8(a) || b.scalar_type() != at::kFloat8_e4m3fn) return Tensor();
  const int ar = trans_a ? 1 : 0, ak = 1 - ar, br = trans_b ? 0 : 1, bk = 1 - br;
  const int64_t M = a.size(ar), K = a.size(ak), N = b.size(br), KB = div_up(K, 128);
  if (M == 0 || N == 0 || K == 0 || K > fp8_longest || b.size(bk) != K || as.size(ar) != (a_2d ? div_up(M, 128) : M) || as.size(ak) != KB || bs.size(br) != (b_2d ? div_up(N, 128) : N) || bs.size(bk) != KB)
    return Tensor();
  if (!fp8_readable(a, ar, ak) || !fp8_readable(b, br, bk) || !fp8_scales(as, ar) || !fp8_scales(bs, br)) return Tensor();
  const Tensor c = fp8_result({M, N}, a, dtype);
  alto_mxfp4_fp8_gemm_t p{};
  p.a = a.data_ptr(); p.b = b.data_ptr(); p.a_scales = static_cast<const float*>(as.data_ptr()); p.b_scales = static_cast<const float*>(bs.data_ptr()); p.c = c.data_ptr();
  p.M = M; p.N = N; p.K = K; p.lda = stride_of(a, ar); p.ldb = stride_of(b, br);
  p.a_ss_r = stride_of(as, ar); p.a_ss_k = stride_of(as, ak); p.b_ss_r = stride_of(bs, br); p.b_ss_k = stride_of(bs, bk); p.ldc = N;
  p.a_code = fp8_code(a.scalar_type()); p.a_is_2d = a_2d; p.b_is_2d = b_2d; p.c_dtype = dtype_code(dtype);
  f.ok("alto_mxfp4_fp8_gemm", api.fp8_gemm(&p, current_stream(a)));
  return c;
}
// as blockwise_fp8_grouped_gemm takes them, offsets contiguous
Tensor fp8_grouped_call(Failure& f, const Tensor& a, const Tensor& as, const Tensor& w, const Tensor& ws, const Tensor& offs, bool w_2d, bool trans_weights, at::ScalarType dtype) {
  if (a.dim() != 2 || w.dim() != 3 || as.dim() != 2 || ws.dim() != 3 || !is_fp8(a) || w.scalar_type() != at::kFloat8_e4m3fn) return Tensor();
  const int wr = trans_weights ? 1 : 2, wk = 3 - wr;
  const int64_t M = a.size(0), K = a.size(1), E = w.size(0), N = w.size(wr), KB = div_up(K, 128);
  if (M == 0 || N == 0 || K == 0 || K > fp8_longest || w.size(wk) != K || offs.size(0) != E + 1 || as.size(0) != M || as.size(1) != KB || ws.size(0) != E || ws.size(wr) != (w_2d ? div_up(N, 128) : N) || ws.size(wk) != KB)
    return Tensor();
  if (!fp8_readable(a, 0, 1) || !fp8_readable(w, wr, wk) || !fp8_scales(as, 0) || !fp8_scales(ws, wr)) return Tensor();
  const Tensor c = fp8_result({M, N}, a, dtype);
  alto_mxfp4_fp8_grouped_gemm_t p{};
  p.a = a.data_ptr(); p.w = w.data_ptr(); p.a_scales = static_cast<const float*>(as.data_ptr()); p.w_scales = static_cast<const float*>(ws.data_ptr()); p.c = c.data_ptr();
  p.offs = static_cast<const int32_t*>(offs.data_ptr());
  p.M = M; p.N = N; p.K = K; p.lda = stride_of(a, 0); p.a_ss_r = stride_of(as, 0); p.a_ss_k = stride_of(as, 1); p.w_se = stride_of(w, 0); p.ldw = stride_of(w, wr);
  p.ws_e = stride_of(ws, 0); p.ws_r = stride_of(ws, wr); p.ws_k = stride_of(ws, wk); p.ldc = N;
  p.a_code = fp8_code(a.scalar_type()); p.w_is_2d = w_2d; p.c_dtype = dtype_code(dtype); p.groups = (int)E;
  f.ok("alto_mxfp4_fp8_grouped_gemm", api.fp8_grouped_gemm(&p, current_stream(a)));
  return c;
}
// as blockwise_fp8_grouped_gemm_weights takes them
Tensor fp8_grouped_weights_call(Failure& f, const Tensor& go, const Tensor& gs, const Tensor& x, const Tensor& xs, const Tensor& offs, at::ScalarType dtype) {
  if (go.dim() != 2 || x.dim() != 2 || gs.dim() != 2 || xs.dim() != 2 || !is_fp8(go) || x.scalar_type() != at::kFloat8_e4m3fn) return Tensor();
  const int64_t P = go.size(0), N = go.size(1), K = x.size(1), E = offs.size(0) - 1;
  if (P == 0 || N == 0 || K == 0 || P > fp8_longest || P % 128 != 0 || x.size(0) != P || gs.size(0) != P / 128 || gs.size(1) != N || xs.size(0) != P / 128 || xs.size(1) != K) return Tensor();
  if (!fp8_readable(go, 1, 0) || !fp8_readable(x, 1, 0) || gs.scalar_type() != at::kFloat || xs.scalar_type() != at::kFloat || (N != 1 && gs.stride(1) != 1) || (K != 1 && xs.stride(1) != 1)) return Tensor();
  const Tensor dw = fp8_result({E, N, K}, go, dtype);
  alto_mxfp4_fp8_grouped_gemm_weights_t p{};
  p.go = go.data_ptr(); p.x = x.data_ptr(); p.go_scales = static_cast<const float*>(gs.data_ptr()); p.x_scales = static_cast<const float*>(xs.data_ptr()); p.dw = dw.data_ptr();
  p.offs = static_cast<const int32_t*>(offs.data_ptr());
  p.tokens = P; p.N = N; p.K = K; p.go_ld = stride_of(go, 1); p.x_ld = stride_of(x, 1); p.go_ss = stride_of(gs, 0); p.x_ss = stride_of(xs, 0); p.dw_se = N * K; p.ld_dw = K;
  p.go_code = fp8_code(go.scalar_type()); p.dw_dtype = dtype_code(dtype); p.groups = (int)E;
  f.ok("alto_mxfp4_fp8_grouped_gemm_weights", api.fp8_grouped_gemm_weights(&p, current_stream(go)));
  return dw;
}
template <typename Call>
py::object fp8_product(Call call) {
  Failure f;
  Tensor out;
  {
    py::gil_scoped_release nogil;
    out = call(f);
  }
  f.raise();
  return out.defined() ? py::cast(out) : py::object(py::none());
}
at::ScalarType result_type(bool f32) { return f32 ? at::kFloat : at::kBFloat16; }
py::object fp8_gemm(const Tensor& a, const Tensor& as, const Tensor& b, const Tensor& bs, bool a_2d, bool b_2d, bool trans_a, bool trans_b, bool f32) {
  if (!plain_operands({&a, &as, &b, &bs})) return py::none();
  return fp8_product([&](Failure& f) { return fp8_gemm_call(f, a, as, b, bs, a_2d, b_2d, trans_a, trans_b, result_type(f32)); });
}
py::object fp8_grouped_gemm(const Tensor& a, const Tensor& as, const Tensor& w, const Tensor& ws, const Tensor& offs, bool w_2d, bool trans_weights, bool f32) {
  if (!plain_operands({&a, &as, &w, &ws}) || !is_offsets(offs)) return py::none();
  return fp8_product([&](Failure& f) { return fp8_grouped_call(f, a, as, w, ws, offs, w_2d, trans_weights, result_type(f32)); });
}
py::object fp8_grouped_gemm_weights(const Tensor& go, const Tensor& gs, const Tensor& x, const Tensor& xs, const Tensor& offs, bool f32) {
  if (!plain_operands({&go, &gs, &x, &xs}) || !is_offsets(offs)) return py::none();
  return fp8_product([&](Failure& f) { return fp8_grouped_weights_call(f, go, gs, x, xs, offs, result_type(f32)); });
}

// A node as the interpreter sees it (y.grad_fn): torch's own attributes, with the name and the saved tensors that a Python function's node has.
template <typename Step>
PyObject* node_saved_tensors(PyObject* self, void*) {
  HANDLE_TH_ERRORS
  const auto& node = reinterpret_cast<torch::autograd::THPCppFunction*>(self)->cdata;
  const variable_list saved = static_cast<torch::autograd::CppNode<Step>&>(*node).ctx_.get_saved_variables();
  py::tuple out(saved.size());
  for (size_t i = 0; i < saved.size(); ++i) out[i] = py::cast(saved[i]);
  return out.release().ptr();
  END_HANDLE_TH_ERRORS
}
PyObject* node_name(PyObject* self, PyObject*) { return PyUnicode_FromString(Py_TYPE(self)->tp_name); }

template <typename Step>
void introduce_node(const char* name) {
  static PyTypeObject type;
  static PyGetSetDef saved_tensors = {"saved_tensors", node_saved_tensors<Step>, nullptr, nullptr, nullptr};
  static PyMethodDef name_method = {"name", node_name, METH_NOARGS, nullptr};
  torch::autograd::_initFunctionPyTypeObject(type, name, nullptr, nullptr);
  const py::object getter = py::reinterpret_steal<py::object>(PyDescr_NewGetSet(&type, &saved_tensors));
  const py::object method = py::reinterpret_steal<py::object>(PyDescr_NewMethod(&type, &name_method));
  if (!getter || !method || PyDict_SetItemString(type.tp_dict, "saved_tensors", getter.ptr()) != 0 || PyDict_SetItemString(type.tp_dict, "name", method.ptr()) != 0)
    throw py::error_already_set();
  PyType_Modified(&type);
  torch::autograd::registerCppFunction(typeid(torch::autograd::CppNode<Step>), &type);
}

}  // namespace

PYBIND11_MODULE(alto_mxfp4_host, m) {
  introduce_node<LinearNode>("MXFP4LinearStepBackward");
  introduce_node<GroupedNode>("MXFP4GroupedStepBackward");
  introduce_node<AttentionNode>("MXFP4AttentionFunctionBackward");
  introduce_node<RotaryNode>("RotaryBackward");
  m.def("bind", &bind);
  m.def("quantize", &quantize);
  m.def("dequantize", &dequantize);
  m.def("gemm", &gemm);
  m.def("gemm_packed", &gemm_packed);
  m.def("grouped_packed", &grouped_packed);
  m.def("grouped_dw_packed", &grouped_dw_packed);
  m.def("attend", &attend);
  m.def("attention_gradients", &attention_gradients_py);
  m.def("attention_step", &attention_step);
  m.def("rotary", &rotary);
  m.def("fp8_quantize", &fp8_quantize);
  m.def("fp8_gemm", &fp8_gemm);
  m.def("fp8_grouped_gemm", &fp8_grouped_gemm);
  m.def("fp8_grouped_gemm_weights", &fp8_grouped_gemm_weights);
  m.def("linear_step", &linear_step);
  m.def("linear_saved", &linear_saved);
  m.def("grouped_step", &grouped_step);
  m.def("grouped_saved", &grouped_saved);
  m.def("draw_hadamard", &draw_hadamard);
  // (the rules that linear.py and grouped_gemm.py state as well, for a comparison of the two)
  m.def("packed_gemm_supported", &packed_gemm_supported);
  m.def("grouped_packed_supported", &grouped_packed_supported);
  m.def("grouped_dw_packed_supported", &grouped_dw_packed_supported);
}
