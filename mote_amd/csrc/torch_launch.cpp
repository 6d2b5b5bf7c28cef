// Native launchers of the torch ops: output allocation, argument blocks and the C-ABI calls of the ops whose
// Python bodies did the same through ctypes. A body's allocations, views and argument fields took 18 to
// 25 us of interpreter time a call (the forward 18.0, the backward 25.1), 7.9 and 10.8 here, and a small
// layer's step is paced by them. Dispatch, autograd and fake implementations stay with the Python ops, and
// so do checks of what a call may pass, except the sizes, types and devices of operands whose extent the
// kernel takes from another one: those are compared here. RuntimeError with the library's message
// when a call fails. Host code only; streams come as raw handles.
#include <c10/core/AutogradState.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/extension.h>

#include <array>
#include <climits>
#include <initializer_list>
#include <string>
#include <tuple>
#include <utility>
#include <vector>

#include "../../include/mote_relation.h"

namespace {

using at::Tensor;
using OptTensor = std::optional<Tensor>;

[[noreturn]] void fail(int rc, const char* what) {
  throw std::runtime_error(std::string(what) + " failed (status " + std::to_string(rc) + "): " + mote_last_error());
}
void check(int rc, const char* what) {
  if (rc != MOTE_OK) fail(rc, what);
}

int code(at::ScalarType t) {
  if (t == at::kFloat) return MOTE_F32;
  if (t == at::kBFloat16) return MOTE_BF16;
  throw py::type_error(std::string("Relation kernels take float32 or bfloat16 tensors, got ") + c10::toString(t));
}
int code(const Tensor& t) { return code(t.scalar_type()); }

mote_view view(const Tensor& t) {
  TORCH_CHECK(t.dim() == 4 && t.stride(3) == 1, "last axis must be contiguous");
  return mote_view{t.data_ptr(), t.stride(0), t.stride(1), t.stride(2)};
}
float* fptr(const Tensor& t) { return static_cast<float*>(t.data_ptr()); }
int32_t* iptr(const Tensor& t) { return static_cast<int32_t*>(t.data_ptr()); }

Tensor empty(at::IntArrayRef sizes, const Tensor& like, at::ScalarType dt) {
  return at::empty(sizes, like.options().dtype(dt).memory_format(std::nullopt));
}
// [B, H, T, D] view over new [B, T, H, D] memory
Tensor heads(int64_t B, int64_t T, int64_t H, int64_t D, const Tensor& like, at::ScalarType dt) {
  return empty({B, T, H, D}, like, dt).transpose(1, 2);
}
Tensor bytes(size_t n, const Tensor& like) { return empty({int64_t(n < 16 ? 16 : n)}, like, at::kByte); }
// a small parameter as contiguous fp32 on the operands' device (itself when it is that already)
Tensor f32(const Tensor& t, const Tensor& like) { return t.detach().to(like.device(), at::kFloat).contiguous(); }

// unit stride on the last axis, strides of whole 16-byte chunks and an aligned base, else a copy
Tensor aligned(const Tensor& t) {
  const int64_t epc = 16 / t.element_size();
  bool ok = t.stride(-1) == 1 && reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0;
  for (int64_t i = 0; i + 1 < t.dim(); ++i) ok = ok && t.stride(i) % epc == 0;
  return ok ? t : t.contiguous();
}
Tensor unit(const Tensor& t) { return t.stride(-1) == 1 ? t : t.contiguous(); }

std::tuple<Tensor, Tensor, Tensor, Tensor> relation_fwd(Tensor p1, Tensor p2, Tensor info, const Tensor& lam, double tau,
                                                        int64_t q_start, const OptTensor& cu, int64_t max_seqlen,
                                                        int64_t stream) {
  const bool varlen = cu.has_value();  // p1, p2, info are then [1, H, total, D]
  p1 = aligned(p1); p2 = aligned(p2); info = aligned(info);
  const int64_t B = p1.size(0), H = p1.size(1), TQ = p1.size(2), D = p1.size(3), TK = p2.size(2);
  const Tensor lam32 = lam.detach().to(at::kFloat).reshape({1}).contiguous();
  Tensor y = heads(B, TQ, H, D, p1, info.scalar_type());
  Tensor ibar = empty({B, H, TQ, D}, p1, at::kFloat), lse = empty({B, H, TQ}, p1, at::kFloat), g = empty({B, H, TQ}, p1, at::kFloat);
  mote_relation_fwd_args a{};
  a.dtype = code(p1);
  a.B = int(varlen ? cu->numel() - 1 : B); a.H = int(H); a.D = int(D);
  a.TQ = int(varlen ? max_seqlen : TQ); a.TK = int(varlen ? max_seqlen : TK); a.q_start = int(q_start);
  a.tau_s = float(tau);
  a.p1 = view(p1); a.p2 = view(p2); a.info = view(info); a.y = view(y);
  a.ibar = fptr(ibar); a.lse = fptr(lse); a.g = fptr(g); a.lam = fptr(lam32);
  if (varlen) {
    a.cu_seqlens = iptr(*cu);
    a.total_rows = int(TQ);
  }
  // scratch of the key-range pieces or the job counters; held until the launch is queued (the caching
  // allocator orders its reuse)
  Tensor ws;
  const size_t n = mote_relation_fwd_workspace(&a);
  if (n) {
    ws = bytes(n, p1);
    a.workspace = ws.data_ptr();
    a.workspace_bytes = n;
  }
  check(mote_relation_fwd(&a, reinterpret_cast<void*>(stream)), varlen ? "mote_relation_fwd (varlen)" : "mote_relation_fwd");
  return {y, g, ibar, lse};
}

std::tuple<Tensor, Tensor, Tensor, Tensor> relation_bwd(Tensor p1, Tensor p2, Tensor info, Tensor ibar, Tensor lse, Tensor g,
                                                        Tensor dy, double tau, int64_t q_start, bool deterministic,
                                                        int64_t stream) {
  p1 = aligned(p1); p2 = aligned(p2); info = aligned(info);
  dy = aligned(dy.to(p1.scalar_type()));
  ibar = ibar.contiguous(); lse = lse.contiguous(); g = g.contiguous();
  const int64_t B = p1.size(0), H = p1.size(1), TQ = p1.size(2), D = p1.size(3), TK = p2.size(2);
  Tensor dp1 = heads(B, TQ, H, D, p1, p1.scalar_type()), dp2 = heads(B, TK, H, D, p1, p2.scalar_type()),
         dinfo = heads(B, TK, H, D, p1, info.scalar_type()), dlam = empty({}, p1, at::kFloat);
  mote_relation_bwd_args a{};
  a.dtype = code(p1);
  a.B = int(B); a.H = int(H); a.TQ = int(TQ); a.TK = int(TK); a.D = int(D); a.q_start = int(q_start);
  a.tau_s = float(tau);
  a.deterministic = deterministic;
  a.p1 = view(p1); a.p2 = view(p2); a.info = view(info); a.dy = view(dy);
  a.ibar = fptr(ibar); a.lse = fptr(lse); a.g = fptr(g);
  a.dp1 = view(dp1); a.dp2 = view(dp2); a.dinfo = view(dinfo);
  a.dlam = fptr(dlam);
  // a step that leaves too little memory for the stored dU runs without it
  const size_t full = mote_relation_bwd_workspace(&a), least = mote_relation_bwd_workspace_min(&a);
  Tensor ws;
  try {
    ws = bytes(full, p1);
  } catch (const c10::OutOfMemoryError&) {
    if (least == full) throw;
    ws = bytes(least, p1);
  }
  a.workspace = ws.data_ptr();
  a.workspace_bytes = size_t(ws.numel());
  check(mote_relation_bwd(&a, reinterpret_cast<void*>(stream)), "mote_relation_bwd");
  return {dp1, dp2, dinfo, dlam};
}

std::tuple<Tensor, Tensor, Tensor> rope_givens(Tensor qkv, const OptTensor& inv_freq, const OptTensor& theta, int64_t H,
                                               int64_t parity, int64_t pos0, int64_t stream) {
  qkv = unit(qkv);
  const int64_t B = qkv.size(0), T = qkv.size(1), D = qkv.size(2) / (3 * H);
  Tensor p1 = heads(B, T, H, D, qkv, qkv.scalar_type()), p2 = heads(B, T, H, D, qkv, qkv.scalar_type()),
         info = heads(B, T, H, D, qkv, qkv.scalar_type());
  Tensor inv, th;
  if (inv_freq) inv = f32(*inv_freq, qkv);
  if (theta) th = f32(*theta, qkv);
  mote_rope_givens_args a{};
  a.dtype = code(qkv);
  a.B = int(B); a.T = int(T); a.H = int(H); a.D = int(D); a.pos0 = int(pos0); a.layer_parity = int(parity);
  a.inv_freq = inv_freq ? fptr(inv) : nullptr;
  a.theta = theta ? fptr(th) : nullptr;
  a.qkv = qkv.data_ptr(); a.qkv_sb = qkv.stride(0); a.qkv_sr = qkv.stride(1);
  a.p1 = view(p1); a.p2 = view(p2); a.info = view(info);
  check(mote_rope_givens_fwd(&a, reinterpret_cast<void*>(stream)), "mote_rope_givens_fwd");
  return {p1, p2, info};
}

std::tuple<Tensor, Tensor> rope_givens_bwd(const Tensor& dp1_, const Tensor& dp2_, const Tensor& dinfo_, Tensor qkv,
                                           const OptTensor& inv_freq, const OptTensor& theta, int64_t H, int64_t parity,
                                           int64_t pos0, bool info_only, int64_t stream) {
  const int64_t B = qkv.size(0), T = qkv.size(1), D = info_only ? qkv.size(2) / H : qkv.size(2) / (3 * H), D3 = 3 * H * D;
  qkv = unit(qkv);
  const at::ScalarType dt = qkv.scalar_type();
  auto grad = [&](const Tensor& t) { return t.stride(-1) == 1 ? t.to(dt) : t.to(dt).contiguous(); };
  const Tensor dp1 = grad(dp1_), dp2 = grad(dp2_), dinfo = grad(dinfo_);
  Tensor dqkv = empty({B, T, D3}, qkv, dt);
  // written whole by the kernel when theta is given
  Tensor dtheta = empty({H / 2 > 1 ? H / 2 : 1}, qkv, at::kFloat);
  if (!theta) dtheta.zero_();
  Tensor inv, th;
  if (inv_freq) inv = f32(*inv_freq, qkv);
  if (theta) th = f32(*theta, qkv);
  mote_rope_givens_bwd_args a{};
  a.dtype = code(qkv);
  a.B = int(B); a.T = int(T); a.H = int(H); a.D = int(D); a.pos0 = int(pos0); a.layer_parity = int(parity);
  a.inv_freq = inv_freq ? fptr(inv) : nullptr;
  a.theta = theta ? fptr(th) : nullptr;
  a.qkv = qkv.data_ptr(); a.qkv_sb = qkv.stride(0); a.qkv_sr = qkv.stride(1);
  a.qkv_info_only = info_only;
  a.dp1 = view(dp1); a.dp2 = view(dp2); a.dinfo = view(dinfo);
  a.dqkv = dqkv.data_ptr(); a.dqkv_sb = dqkv.stride(0); a.dqkv_sr = dqkv.stride(1);
  a.dtheta = fptr(dtheta);
  const Tensor ws = bytes(mote_rope_givens_bwd_workspace(&a), qkv);
  a.workspace = ws.data_ptr();
  a.workspace_bytes = size_t(ws.numel());
  check(mote_rope_givens_bwd(&a, reinterpret_cast<void*>(stream)), "mote_rope_givens_bwd");
  return {dqkv, dtheta};
}

Tensor linear_wgrad(Tensor a_, Tensor x, at::ScalarType dtype, int64_t stream) {
  TORCH_CHECK(a_.dim() == 2 && x.dim() == 2 && a_.size(0) == x.size(0) && a_.scalar_type() == x.scalar_type() &&
                  a_.device() == x.device(),
              "linear_wgrad: a [M, N] and x [M, K] of one dtype and device, got ", a_.sizes(), " ", a_.scalar_type(), " and ",
              x.sizes(), " ", x.scalar_type());
  // rows the kernel can walk: apart (an expanded gradient has stride 0), within its 32-bit offsets, aligned
  auto rows = [](const Tensor& t) {
    const int64_t sr = t.stride(0);
    const bool ok = t.stride(1) == 1 && sr >= t.size(1) && sr < (int64_t(1) << 24) && sr % 8 == 0 &&
                    reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0;
    return ok ? t : t.clone(at::MemoryFormat::Contiguous);  // (contiguous() keeps a contiguous tensor off a boundary)
  };
  a_ = rows(a_);
  x = rows(x);
  Tensor dw = empty({a_.size(1), x.size(1)}, a_, dtype);
  mote_linear_wgrad_args a{};
  a.dtype = code(a_); a.dw_dtype = code(dw);
  a.M = int(a_.size(0)); a.N = int(a_.size(1)); a.K = int(x.size(1));
  a.a = a_.data_ptr(); a.a_sr = a_.stride(0);
  a.x = x.data_ptr(); a.x_sr = x.stride(0);
  a.dw = dw.data_ptr(); a.dw_sr = dw.stride(0);
  const Tensor ws = bytes(mote_linear_wgrad_workspace(&a), a_);
  a.workspace = ws.data_ptr();
  a.workspace_bytes = size_t(ws.numel());
  check(mote_linear_wgrad(&a, reinterpret_cast<void*>(stream)), "mote_linear_wgrad");
  return dw;
}

// [..., D] -> [rows, D] with unit element stride (a view when possible)
Tensor rows2d(const Tensor& t_) { return unit(t_).reshape({-1, t_.size(-1)}); }

// (y, s or an empty stand-in when s is x itself, rstd); s_dtype: the summed stream's type
std::tuple<Tensor, Tensor, Tensor> add_rms_norm(const Tensor& x, const Tensor& weight, const OptTensor& residual, double eps,
                                                at::ScalarType s_dtype, int64_t stream) {
  const int64_t D = x.size(-1);
  const Tensor x2 = rows2d(x), w = f32(weight, x);
  const int64_t rows = x2.size(0);
  Tensor r2;
  if (residual) r2 = rows2d(*residual);
  Tensor y = empty(x.sizes(), x, x.scalar_type());
  const bool sum = residual.has_value() || s_dtype != x.scalar_type();
  Tensor s = sum ? empty(x.sizes(), x, s_dtype) : empty({0}, x, x.scalar_type());
  Tensor rstd = empty({rows}, x, at::kFloat);
  mote_add_rms_norm_args a{};
  a.dtype = code(x2); a.out_dtype = code(y);
  a.res_dtype = residual ? code(r2) : a.dtype;
  a.res_out_dtype = sum ? code(s) : a.dtype;
  a.rows = int(rows); a.D = int(D); a.eps = float(eps);
  a.x = x2.data_ptr(); a.x_sr = x2.stride(0);
  if (residual) {
    a.residual = r2.data_ptr();
    a.res_sr = r2.stride(0);
  }
  a.weight = fptr(w);
  a.y = y.data_ptr(); a.y_sr = D;
  if (sum) {
    a.residual_out = s.data_ptr();
    a.res_out_sr = D;
  }
  a.rstd = fptr(rstd);
  check(mote_add_rms_norm_fwd(&a, reinterpret_cast<void*>(stream)), "mote_add_rms_norm_fwd");
  return {y, s, rstd};
}

std::tuple<Tensor, Tensor, Tensor> add_rms_norm_bwd(const Tensor& dy, const OptTensor& dres_out, const Tensor& s, const Tensor& rstd,
                                                    const Tensor& weight, at::ScalarType x_dtype, bool has_res,
                                                    at::ScalarType res_dtype, int64_t stream) {
  const int64_t D = s.size(-1);
  const Tensor dy2 = rows2d(dy), s2 = rows2d(s), w = f32(weight, s);
  Tensor dro2;
  if (dres_out) dro2 = rows2d(*dres_out);
  Tensor dx = empty(s.sizes(), s, x_dtype);
  Tensor dres = has_res ? empty(s.sizes(), s, res_dtype) : empty({0}, s, res_dtype);
  Tensor dw = empty({D}, s, at::kFloat);
  mote_add_rms_norm_bwd_args a{};
  a.dtype = code(dy2); a.s_dtype = code(s2); a.dx_dtype = code(dx);
  a.dres_out_dtype = dres_out ? code(dro2) : a.dtype;
  a.dres_dtype = has_res ? code(dres) : a.dtype;
  a.rows = int(s2.size(0)); a.D = int(D);
  a.dy = dy2.data_ptr(); a.dy_sr = dy2.stride(0);
  if (dres_out) {
    a.dres_out = dro2.data_ptr();
    a.dres_out_sr = dro2.stride(0);
  }
  a.s = s2.data_ptr(); a.s_sr = s2.stride(0);
  a.rstd = fptr(rstd); a.weight = fptr(w);
  a.dx = dx.data_ptr(); a.dx_sr = D;
  if (has_res) {
    a.dresidual = dres.data_ptr();
    a.dres_sr = D;
  }
  a.dweight = fptr(dw);
  const Tensor ws = bytes(mote_add_rms_norm_bwd_workspace(&a), s);
  a.workspace = ws.data_ptr();
  a.workspace_bytes = size_t(ws.numel());
  check(mote_add_rms_norm_bwd(&a, reinterpret_cast<void*>(stream)), "mote_add_rms_norm_bwd");
  return {dx, dres, dw};
}

// The fused prologue; ws: the stacked weight, or the three (p1, p2, I~ projections); p2 / info: views to
// write instead of new tensors. The kernel reads its operands at the sizes that x and H give: they are checked
// against those here (a longer stack, frequency or angle tensor is read at its start). The cos / sin table (memoised by the caller) comes as `table`.
std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor> qkv_rope(const Tensor& x, const std::vector<Tensor>& ws, const OptTensor& inv_freq,
                                                            const OptTensor& theta, int64_t H, int64_t parity, int64_t pos0,
                                                            bool keep_info, const OptTensor& norm_w1, const OptTensor& norm_w2,
                                                            double eps, const Tensor& table, bool table_ready, const OptTensor& p2_,
                                                            const OptTensor& info_, int64_t stream) {
  const int64_t B = x.size(0), T = x.size(1), K = x.size(2), D = K / H;
  const at::ScalarType dt = x.scalar_type();
  TORCH_CHECK(dt == at::kBFloat16 && K == H * D && x.is_contiguous(), "qkv_rope: x must be bf16 of ", H, " heads, got ", dt, " rows of ", K);
  for (const Tensor& w : ws)
    TORCH_CHECK(w.dim() == 2 && (ws.size() == 3 ? w.size(0) == K : w.size(0) >= 3 * K) && w.size(1) == K &&
                    w.scalar_type() == dt && w.device() == x.device() && w.is_contiguous(),
                "qkv_rope: weights must be contiguous bf16 [", K, ", ", K, "] each or [", 3 * K, ", ", K, "] stacked, on x's device");
  TORCH_CHECK(!inv_freq || inv_freq->numel() >= D / 2, "qkv_rope: inv_freq needs ", D / 2, " values");
  TORCH_CHECK(!theta || theta->numel() >= H / 2, "qkv_rope: theta needs ", H / 2, " values");
  for (const OptTensor* t : {&p2_, &info_})  // the caller's memory: the kernel writes all of [B, H, T, D]
    TORCH_CHECK(!t->has_value() || ((*t)->sizes() == at::IntArrayRef({B, H, T, D}) && (*t)->scalar_type() == dt &&
                                    (*t)->device() == x.device()),
                "qkv_rope: P2 and I~ must be [", B, ", ", H, ", ", T, ", ", D, "] in x's dtype on x's device");
  Tensor p1 = heads(B, T, H, D, x, dt);
  Tensor p2 = p2_ ? *p2_ : heads(B, T, H, D, x, dt), info = info_ ? *info_ : heads(B, T, H, D, x, dt);
  const bool norm = norm_w1.has_value();
  Tensor iraw = keep_info ? empty({B, T, K}, x, dt) : empty({0}, x, dt);
  Tensor qkraw = keep_info && norm ? empty({B, T, 2 * K}, x, dt) : empty({0}, x, dt);
  mote_qkv_rope_args a{};
  a.B = int(B); a.T = int(T); a.H = int(H); a.D = int(D); a.pos0 = int(pos0); a.layer_parity = int(parity);
  a.x = x.data_ptr(); a.x_sb = T * K; a.x_sr = K;  // contiguous (the strides of axes of one element may be any)
  a.w = ws[0].data_ptr(); a.w_sr = K;
  Tensor inv, th, n1, n2;
  if (inv_freq) {
    inv = f32(*inv_freq, x);
    a.inv_freq = fptr(inv);
  }
  if (theta) {
    th = f32(*theta, x);
    a.theta = fptr(th);
  }
  a.p1 = view(p1); a.p2 = view(p2); a.info = view(info);
  if (keep_info) {
    a.info_raw = iraw.data_ptr(); a.ir_sb = iraw.stride(0); a.ir_sr = iraw.stride(1);
  }
  if (norm) {
    n1 = f32(*norm_w1, x);
    n2 = f32(*norm_w2, x);
    a.norm_w1 = fptr(n1); a.norm_w2 = fptr(n2); a.norm_eps = float(eps);
    if (keep_info) {
      a.qk_raw = qkraw.data_ptr(); a.qr_sb = qkraw.stride(0); a.qr_sr = qkraw.stride(1);
    }
  }
  a.workspace = table.data_ptr(); a.workspace_bytes = size_t(table.numel()); a.table_ready = table_ready;
  void* st = reinterpret_cast<void*>(stream);
  if (ws.size() == 3) check(mote_qkv_rope_parts_fwd(&a, ws[1].data_ptr(), ws[2].data_ptr(), st), "mote_qkv_rope_parts_fwd");
  else check(mote_qkv_rope_fwd(&a, st), "mote_qkv_rope_fwd");
  return {p1, p2, info, iraw, qkraw};
}

std::tuple<Tensor, Tensor, Tensor, Tensor> chunk_route(const Tensor& m, int64_t stream) {
  const int64_t B = m.size(0), L = m.size(1);
  Tensor cum = empty({B, L}, m, at::kInt), perm = empty({B, L}, m, at::kInt), num = empty({B}, m, at::kInt),
         cu = empty({B + 1}, m, at::kInt);
  mote_chunk_route_args a{};
  a.B = int(B); a.L = int(L);
  a.mask = static_cast<const uint8_t*>(m.data_ptr()); a.mask_sr = m.stride(0);
  a.cum = iptr(cum); a.perm = iptr(perm); a.num = iptr(num); a.cu_seqlens = iptr(cu);
  if (B == 0) cu.zero_();
  check(mote_chunk_route(&a, reinterpret_cast<void*>(stream)), "mote_chunk_route");
  return {cum, perm, num, cu};
}

std::tuple<Tensor, Tensor> dechunk(const Tensor& h, const Tensor& pr, const Tensor& perm, const Tensor& num, const Tensor& cum,
                                   int64_t L, double eps, const OptTensor& init, int64_t stream) {
  const int64_t B = h.size(0), M = h.size(1), D = h.size(2);
  Tensor out = empty({B, L, D}, h, h.scalar_type()), w = empty({B, M, D}, h, at::kFloat), ini;
  if (init) ini = f32(*init, h);
  mote_dechunk_args a{};
  a.dtype = code(h); a.prob_dtype = code(pr); a.out_dtype = a.dtype;
  a.B = int(B); a.L = int(L); a.M = int(M); a.D = int(D); a.eps = float(eps);
  a.hidden = h.data_ptr(); a.h_sb = h.stride(0); a.h_sr = h.stride(1);
  a.prob = pr.data_ptr(); a.p_sb = pr.stride(0); a.p_sr = pr.stride(1);
  a.perm = iptr(perm); a.num = iptr(num); a.cum = iptr(cum);
  a.init = init ? fptr(ini) : nullptr;
  a.out = out.data_ptr(); a.o_sb = out.stride(0); a.o_sr = out.stride(1);
  a.w = fptr(w);
  const Tensor ws = bytes(mote_dechunk_workspace(&a), h);
  a.workspace = ws.data_ptr();
  a.workspace_bytes = size_t(ws.numel());
  check(mote_dechunk_fwd(&a, reinterpret_cast<void*>(stream)), "mote_dechunk_fwd");
  return {out, w};
}

std::tuple<Tensor, Tensor> dechunk_bwd(const Tensor& g, const Tensor& h, const Tensor& pr, const Tensor& perm, const Tensor& num,
                                       const Tensor& m, const Tensor& cum, const Tensor& w, double eps, int64_t stream) {
  const int64_t B = h.size(0), M = h.size(1), D = h.size(2), L = g.size(1);
  Tensor dh = empty({B, M, D}, h, h.scalar_type()), dp = empty({B, L, 2}, h, pr.scalar_type());
  mote_dechunk_bwd_args a{};
  a.dtype = code(h); a.prob_dtype = code(pr); a.dout_dtype = code(g); a.dx_dtype = code(dh); a.dprob_dtype = code(dp);
  a.B = int(B); a.L = int(L); a.M = int(M); a.D = int(D); a.eps = float(eps);
  a.dout = g.data_ptr(); a.g_sb = g.stride(0); a.g_sr = g.stride(1);
  a.hidden = h.data_ptr(); a.h_sb = h.stride(0); a.h_sr = h.stride(1);
  a.prob = pr.data_ptr(); a.p_sb = pr.stride(0); a.p_sr = pr.stride(1);
  a.perm = iptr(perm); a.num = iptr(num);
  a.mask = static_cast<const uint8_t*>(m.data_ptr()); a.mask_sr = m.stride(0);
  a.cum = iptr(cum); a.w = fptr(w);
  a.dhidden = dh.data_ptr(); a.dh_sb = dh.stride(0); a.dh_sr = dh.stride(1);
  a.dprob = dp.data_ptr(); a.dp_sb = dp.stride(0); a.dp_sr = dp.stride(1);
  const Tensor ws = bytes(mote_dechunk_bwd_workspace(&a), h);
  a.workspace = ws.data_ptr();
  a.workspace_bytes = size_t(ws.numel());
  check(mote_dechunk_bwd(&a, reinterpret_cast<void*>(stream)), "mote_dechunk_bwd");
  return {dh, dp};
}

// ---- the cache in 4 bits and the 8-bit products ----------------------------------------------------------
// Checks, allocation and launch in one call, on the operands' device and its current stream: a step of a
// token is paced by its calls (with the stream and a device context taken in Python a call of a decode step
// took 5.8 us of host time, 5.0 so).
template <typename... A>
[[noreturn]] void bad_value(A&&... a) { throw py::value_error(c10::str(std::forward<A>(a)...)); }
void on_gpu(const Tensor& t, const char* what) {
  if (!t.is_cuda()) throw std::runtime_error(c10::str(what, " needs the HIP library and an MI355X"));
}
// the operands' device as the current one for the life of the object, and its current stream
struct On {
  c10::DeviceGuard guard;
  void* stream;
  explicit On(const Tensor& t) : guard(t.device()), stream(c10::hip::getCurrentHIPStream(t.device().index()).stream()) {}
};
// Refuses tensors, parameters and given outputs among them, whose derivative would be lost: tangents of forward
// mode (which no_grad leaves on), gradients under grad mode.
void no_tangent(const char* what, std::initializer_list<const Tensor*> ts) {
  if (!c10::AutogradState::get_tls_state().get_fw_grad_mode()) return;
  for (const Tensor* t : ts)
    if (t->_fw_grad(0).defined()) throw std::runtime_error(c10::str(what, " has no forward-mode derivative: it takes no dual tensors"));
}
void no_grad(const char* what, std::initializer_list<const Tensor*> ts) {
  no_tangent(what, ts);
  if (!at::GradMode::is_enabled()) return;
  for (const Tensor* t : ts)
    if (t->requires_grad()) throw std::runtime_error(c10::str(what, " has no backward: call it under torch.no_grad()"));
}
// Refuses a result that lies over an operand: it would be written while another workgroup still reads there.
// Both are rows of `width` elements back to back within, `stride` apart; columns of one buffer (the same stride,
// the columns apart) pass.
void apart(const Tensor& out, int64_t out_width, const Tensor& in, int64_t in_width, int64_t rows, const char* what) {
  const int64_t e = out.element_size(), so = rows > 1 ? out.stride(0) : 0, si = rows > 1 ? in.stride(0) : 0;
  const int64_t o = reinterpret_cast<int64_t>(out.data_ptr()) / e, i = reinterpret_cast<int64_t>(in.data_ptr()) / e;
  if (rows == 0 || o >= i + (rows - 1) * si + in_width || i >= o + (rows - 1) * so + out_width) return;
  if (rows > 1 && so == si) {
    const int64_t d = ((o - i) % so + so) % so;
    if (d >= in_width && d + out_width <= so) return;
  }
  bad_value(what, ": the output lies over an input");
}
// Whether every element of a view has an address of its own: taken by stride, a step passes all that the smaller
// ones reach. With `other`, a view of as many dims and the same sizes, whether two views that are separate each are
// so together (as one view with a dim of two more where their strides agree, by the ranges that they span where not).
bool separate(const Tensor& t, const Tensor* other = nullptr) {
  if (t.numel() == 0 || (!other && t.is_contiguous())) return true;
  constexpr int kMost = 8;
  std::array<std::pair<int64_t, int64_t>, kMost + 1> dim;  // stride, size
  int n = 0;
  bool alike = true;
  int64_t span = 1, span2 = 1;
  for (int64_t i = 0; i < t.dim() && n < kMost; ++i) {
    if (t.size(i) == 1) continue;
    dim[n++] = {t.stride(i), t.size(i)};
    span += (t.size(i) - 1) * t.stride(i);
    if (other) {
      alike = alike && other->stride(i) == t.stride(i);
      span2 += (other->size(i) - 1) * other->stride(i);
    }
  }
  if (other) {
    const int64_t e = t.element_size(), a = reinterpret_cast<int64_t>(t.data_ptr()), b = reinterpret_cast<int64_t>(other->data_ptr());
    if (b >= a + span * e || a >= b + span2 * e) return true;
    if (!alike || (b - a) % e) return false;
    dim[n++] = {b > a ? (b - a) / e : (a - b) / e, 2};
  }
  for (int i = 1; i < n; ++i)
    for (int j = i; j > 0 && dim[j] < dim[j - 1]; --j) std::swap(dim[j], dim[j - 1]);
  int64_t reach = 1;
  for (int i = 0; i < n; ++i) {
    if (dim[i].first < reach) return false;
    reach += dim[i].first * (dim[i].second - 1);
  }
  return true;
}
// whether the ranges of memory that two views span are apart
bool ranges_apart(const Tensor& a, const Tensor& b) {
  auto end = [](const Tensor& t) {
    int64_t span = 1;
    for (int64_t i = 0; i < t.dim(); ++i) span += (t.size(i) - 1) * t.stride(i);
    return reinterpret_cast<int64_t>(t.data_ptr()) + span * t.element_size();
  };
  if (a.numel() == 0 || b.numel() == 0) return true;
  return reinterpret_cast<int64_t>(a.data_ptr()) >= end(b) || reinterpret_cast<int64_t>(b.data_ptr()) >= end(a);
}
// an int64 position per sequence (read, and with `advance` written, by the kernel as it is)
void positions(const Tensor& t, int64_t B, c10::Device dev, const char* what, const char* name) {
  if (t.scalar_type() != at::kLong || t.device() != dev || t.numel() != B || !t.is_contiguous())
    bad_value(what, ": ", name, " must be a contiguous int64 tensor of B = ", B, " on the rows' device");
}

struct Cache4 {
  mote_cache4 c;
  int64_t capacity;
};
Cache4 cache4(const Tensor& p2, const Tensor& s2, const Tensor& info, const Tensor& si, int64_t B, int64_t H, int64_t D,
              c10::Device dev, bool writes, const char* what) {
  if (D <= 0 || D > 128 || D % 8) bad_value(what, ": head dim ", D, " unsupported (need 8 <= D <= 128, D % 8 == 0)");
  if (B > INT_MAX || H > INT_MAX) bad_value(what, ": ", B, " sequences of ", H, " heads (sizes beyond 32 bits)");
  const int64_t G = (D + 31) / 32;
  const int64_t cap = p2.dim() == 4 ? p2.size(2) : 0;
  auto check = [&](const Tensor& t, const Tensor& like, int64_t width, at::ScalarType dt, const char* name) {
    if (t.dim() != 4 || t.size(0) != B || t.size(1) != H || t.size(2) != cap || t.size(3) != width || cap < 1)
      bad_value(what, ": ", name, " must be [B, H, capacity, ", width, "] = [", B, ", ", H, ", ", cap, ", ", width, "], got ", t.sizes());
    if (t.scalar_type() != dt || t.device() != dev)
      throw py::type_error(c10::str(what, ": ", name, " must be ", c10::toString(dt), " on the rows' device"));
    if ((width > 1 && t.stride(3) != 1) || (cap > 1 && t.stride(2) != width))
      bad_value(what, ": the rows of a head must lie back to back (", name, ")");
    for (int d = 0; d < 2; ++d) {
      if (t.size(d) > 1 && t.stride(d) != like.stride(d)) bad_value(what, ": P2 and I~ must have the same strides");
    }
    // heads (or sequences) that share rows would be written over one another
    if (writes && !separate(t)) bad_value(what, ": ", name, " holds its rows for several heads at once");
  };
  check(p2, p2, 16 * G, at::kByte, "the codes of P2");
  check(info, p2, 16 * G, at::kByte, "the codes of I~");
  check(s2, s2, G, at::kBFloat16, "the scales of P2");
  check(si, s2, G, at::kBFloat16, "the scales of I~");
  if (writes && (!separate(p2, &info) || !separate(s2, &si))) bad_value(what, ": P2 and I~ must not be the same rows");
  Cache4 r;
  r.c = mote_cache4{p2.data_ptr(), s2.data_ptr(), info.data_ptr(), si.data_ptr(),
                    p2.size(0) > 1 ? p2.stride(0) : 0, p2.size(1) > 1 ? p2.stride(1) : 0,
                    s2.size(0) > 1 ? s2.stride(0) : 0, s2.size(1) > 1 ? s2.stride(1) : 0};
  r.capacity = cap;
  if (cap > (int64_t(1) << 30)) bad_value(what, ": a capacity of ", cap, " rows (at most 2^30)");
  return r;
}

void rows_of_start(mote_cache4_rows_args& a, const Cache4& c, int64_t start, const OptTensor& start_dev, const OptTensor& lens,
                   int64_t B, int64_t T, c10::Device dev, const char* what) {
  if (T > INT_MAX) bad_value(what, ": ", T, " rows (sizes beyond 32 bits)");
  if (start_dev) {
    positions(*start_dev, B, dev, what, "start");
    a.start_dev = static_cast<const int64_t*>(start_dev->data_ptr());
  } else if (start < 0 || T < 0 || start > c.capacity - T) {
    throw std::runtime_error(c10::str(what, ": rows ", start, " to ", start + T, " in a capacity of ", c.capacity));
  }
  a.start = start;
  if (lens) {
    positions(*lens, B, dev, what, "lens");
    a.lens = static_cast<const int64_t*>(lens->data_ptr());
  }
  a.cache = c.c;
  a.capacity = int(c.capacity);
}

void cache4_write(const Tensor& k, const Tensor& ks, const Tensor& v, const Tensor& vs, Tensor p2, Tensor info, int64_t start,
                  const OptTensor& start_dev, const OptTensor& lens) {
  const char* what = "cache4_write";
  if (p2.dim() != 4 || info.sizes() != p2.sizes()) bad_value(what, ": p2 and info must both be [B, H, T, D]");
  if (info.scalar_type() != p2.scalar_type() || info.device() != p2.device())
    throw py::type_error("cache4_write: p2 and info must share a dtype and a device");
  const int64_t B = p2.size(0), H = p2.size(1), T = p2.size(2), D = p2.size(3);
  const Cache4 c = cache4(k, ks, v, vs, B, H, D, p2.device(), true, what);
  mote_cache4_rows_args a{};
  a.dtype = code(p2);
  rows_of_start(a, c, start, start_dev, lens, B, T, p2.device(), what);
  no_grad(what, {&p2, &info});
  on_gpu(p2, what);
  const On on(p2);
  p2 = aligned(p2); info = aligned(info);
  a.B = int(B); a.H = int(H); a.T = int(T); a.D = int(D);
  a.p2 = view(p2); a.info = view(info);
  check(mote_cache4_write(&a, on.stream), "mote_cache4_write");
}

std::tuple<Tensor, Tensor> cache4_read(const Tensor& k, const Tensor& ks, const Tensor& v, const Tensor& vs, int64_t D,
                                       int64_t start, const OptTensor& start_dev, int64_t rows, at::ScalarType dtype,
                                       const OptTensor& out2, const OptTensor& outi) {
  const char* what = "cache4_read";
  if (k.dim() != 4) bad_value(what, ": the codes of P2 must be [B, H, capacity, 16 G]");
  const int64_t B = k.size(0), H = k.size(1);
  const Cache4 c = cache4(k, ks, v, vs, B, H, D, k.device(), false, what);
  mote_cache4_rows_args a{};
  if (rows < 0) bad_value(what, ": ", rows, " rows");
  rows_of_start(a, c, start, start_dev, std::nullopt, B, rows, k.device(), what);
  Tensor p2, info;
  if (out2) {
    p2 = *out2; info = *outi;
    for (const Tensor* t : {&p2, &info}) {
      if (t->dim() != 4 || t->size(0) != B || t->size(1) != H || t->size(2) != rows || t->size(3) != D || t->device() != k.device())
        bad_value(what, ": out must be two [B, H, rows, D] tensors on the cache's device");
      if (!separate(*t)) bad_value(what, ": out holds its rows for several places at once");
      for (const Tensor* held : {&k, &ks, &v, &vs})
        if (!ranges_apart(*t, *held)) bad_value(what, ": out lies over the cache");
    }
    if (!separate(p2, &info)) bad_value(what, ": the two tensors of out lie over one another");
    if (info.scalar_type() != p2.scalar_type()) throw py::type_error("cache4_read: out must be two tensors of one dtype");
    if (p2.requires_grad() || info.requires_grad()) throw std::runtime_error("cache4_read: out must not require a gradient");
    no_tangent(what, {&p2, &info});
  }
  a.dtype = code(out2 ? p2.scalar_type() : dtype);
  on_gpu(k, what);
  const On on(k);
  if (!out2) {
    p2 = empty({B, H, rows, D}, k, dtype);
    info = empty({B, H, rows, D}, k, dtype);
  }
  a.B = int(B); a.H = int(H); a.T = int(rows); a.D = int(D);
  a.p2 = view(p2); a.info = view(info);
  check(mote_cache4_read(&a, on.stream), "mote_cache4_read");
  return {p2, info};
}

// a small fp32 parameter of n values on `like`'s device (itself when it is that already)
Tensor small_f32(const Tensor& t, int64_t n, const Tensor& like, const char* what, const char* name) {
  if (t.numel() != n || t.device() != like.device())
    bad_value(what, ": ", name, " must be a tensor of ", n, " element(s) on the inputs' device");
  return t.scalar_type() == at::kFloat && t.is_contiguous() ? t : t.detach().to(at::kFloat).contiguous();
}
void check_run(const OptTensor& run, const Tensor& like, const char* what) {
  if (run && ((run->scalar_type() != at::kBool && run->scalar_type() != at::kByte) || run->numel() != 1 || run->device() != like.device()))
    bad_value(what, ": run must be a one-element bool or uint8 tensor on the inputs' device");
}

std::tuple<Tensor, Tensor> relation_decode4(const Tensor& p1, const Tensor& p2, const Tensor& info, const Tensor& S, const Tensor& k,
                                            const Tensor& ks, const Tensor& v, const Tensor& vs, const Tensor& lam, double tau,
                                            const OptTensor& inv_freq, const OptTensor& theta, int64_t layer_idx, bool advance,
                                            const OptTensor& workspace, const OptTensor& y_, const OptTensor& g_, const OptTensor& xm,
                                            const OptTensor& run, bool rope_f32) {
  const char* what = "relation_decode4";
  if (p1.dim() != 3) bad_value(what, ": p1/p2/info must be [B, H, dh]");
  const int64_t B = p1.size(0), H = p1.size(1), D = p1.size(2);
  const c10::Device dev = p1.device();
  for (const Tensor* t : {&p1, &p2, &info}) {
    if (t->sizes() != p1.sizes() || t->stride(2) != 1 || t->stride(1) != D || (B > 1 && t->stride(0) != p1.stride(0)))
      bad_value(what, ": p1/p2/info must be [B, H, dh] with head stride dh and one batch stride");
    if (t->scalar_type() != p1.scalar_type() || t->device() != dev)
      throw py::type_error("relation_decode4: p1, p2 and info must share a dtype and a device");
  }
  if (B < 1 || H < 1 || H % 2) bad_value(what, ": B = ", B, " sequences of H = ", H, " heads (an even number)");
  mote_relation_decode4_args a{};
  a.dtype = code(p1);
  const Cache4 c = cache4(k, ks, v, vs, B, H, D, dev, true, what);
  positions(S, B, dev, what, "S");
  const Tensor lam32 = small_f32(lam, 1, p1, what, "lam");
  Tensor inv, th;
  if (inv_freq) inv = small_f32(*inv_freq, D / 2, p1, what, "inv_freq");
  if (theta) th = small_f32(*theta, H / 2, p1, what, "theta");
  if (xm && (xm->scalar_type() != at::kFloat || xm->numel() != B || !xm->is_contiguous() || xm->device() != dev))
    bad_value(what, ": xm must be a contiguous fp32 tensor of B elements");
  check_run(run, p1, what);
  if (workspace && (workspace->device() != dev || !workspace->is_contiguous()))
    bad_value(what, ": workspace must be a contiguous tensor on the inputs' device");
  if (y_ && (y_->sizes() != p1.sizes() || y_->scalar_type() != p1.scalar_type() || y_->device() != dev || y_->stride(2) != 1 ||
             y_->stride(1) != D || (B > 1 && y_->stride(0) < H * D)))
    bad_value(what, ": y must be [B, H, dh] in the inputs' dtype with head stride dh");
  if (g_ && (g_->dim() != 2 || g_->size(0) != B || g_->size(1) != H || g_->scalar_type() != at::kFloat || g_->device() != dev ||
             !g_->is_contiguous()))
    bad_value(what, ": g must be a contiguous fp32 [B, H] tensor");
  if (y_)
    for (const Tensor* t : {&p1, &p2, &info}) apart(*y_, H * D, *t, H * D, B, what);
  no_grad(what, {&p1, &p2, &info, &lam});
  for (const OptTensor* t : {&inv_freq, &theta, &y_, &g_, &xm})
    if (*t) no_grad(what, {&**t});
  on_gpu(p1, what);
  const On on(p1);
  Tensor y = y_ ? *y_ : empty({B, H, D}, p1, p1.scalar_type());
  Tensor g = g_ ? *g_ : empty({B, H}, p1, at::kFloat);
  a.B = int(B); a.H = int(H); a.D = int(D); a.capacity = int(c.capacity);
  a.layer_parity = int(((layer_idx % 2) + 2) % 2);
  a.flags = (advance ? MOTE_DECODE_ADVANCE : 0) | (rope_f32 ? MOTE_DECODE_ROPE_F32 : 0);
  a.tau_s = float(tau);
  a.lam = fptr(lam32);
  a.inv_freq = inv_freq ? fptr(inv) : nullptr;
  a.theta = theta ? fptr(th) : nullptr;
  a.S = static_cast<int64_t*>(S.data_ptr());
  a.p1 = p1.data_ptr(); a.p2 = p2.data_ptr(); a.info = info.data_ptr(); a.in_sb = p1.stride(0);
  a.cache = c.c;
  a.y = y.data_ptr(); a.y_sb = y.stride(0); a.g = fptr(g);
  const int64_t need = int64_t(mote_relation_decode4_workspace(&a));
  // the halves that counters and partials lie in follow from the bytes: one workspace, one number of them
  if (workspace && workspace->numel() * workspace->element_size() != need)
    bad_value(what, ": a workspace of ", workspace->numel() * workspace->element_size(), " bytes, ", need,
              " needed (decode4_workspace makes one for these sizes)");
  const Tensor ws = workspace ? *workspace : at::zeros({need}, p1.options().dtype(at::kByte));
  a.workspace = ws.data_ptr();
  a.workspace_bytes = size_t(ws.numel()) * ws.element_size();
  a.xm = xm ? fptr(*xm) : nullptr;
  a.run = run ? static_cast<const unsigned char*>(run->data_ptr()) : nullptr;
  check(mote_relation_decode4(&a, on.stream), "mote_relation_decode4");
  return {y, g};
}

std::tuple<Tensor, Tensor> quantize_rows(Tensor x) {
  if (x.dim() != 2 || x.size(1) < 1) bad_value("quantize_rows: x must be [M, K]");
  mote_quantize_rows_args a{};
  a.dtype = code(x);
  no_grad("quantize_rows", {&x});
  on_gpu(x, "quantize_rows");
  const On on(x);
  x = unit(x);
  const int64_t M = x.size(0), K = x.size(1);
  Tensor q = empty({M, (K + 127) / 128 * 128}, x, at::kChar), scale = empty({M}, x, at::kFloat);
  TORCH_CHECK(M <= INT_MAX && K <= INT_MAX, "quantize_rows: sizes beyond 32 bits");
  a.M = int(M); a.K = int(K);
  a.x = x.data_ptr(); a.x_sr = x.stride(0);
  a.q = static_cast<int8_t*>(q.data_ptr()); a.scale = fptr(scale);
  check(mote_quantize_rows(&a, on.stream), "mote_quantize_rows");
  return {q, scale};
}

Tensor int8_linear(const Tensor& x_, const Tensor& wq, const Tensor& ws, int64_t K, const OptTensor& out, const OptTensor& run,
                   const OptTensor& g, const OptTensor& xm) {
  const char* what = "int8_linear";
  if (x_.dim() < 1 || x_.size(-1) != K || K < 1) bad_value(what, ": x must be [..., ", K, "], got ", x_.sizes());
  const int64_t Kp = (K + 127) / 128 * 128;
  if (wq.dim() != 2 || wq.size(0) < 1 || wq.size(1) != Kp || !wq.is_contiguous() || ws.numel() != wq.size(0) || !ws.is_contiguous())
    bad_value(what, ": the weight must be contiguous codes [N, ", Kp, "] with N scales");
  if (wq.scalar_type() != at::kChar || ws.scalar_type() != at::kFloat || wq.device() != x_.device() || ws.device() != x_.device())
    throw py::type_error("int8_linear: the weight must be int8 codes and fp32 scales on x's device");
  const int64_t N = wq.size(0), M = x_.numel() / K;
  mote_int8_linear_args a{};
  a.dtype = code(x_);
  check_run(run, x_, what);
  std::vector<int64_t> sizes = x_.sizes().vec();
  sizes.back() = N;
  if (out && (out->sizes() != at::IntArrayRef(sizes) || out->scalar_type() != x_.scalar_type() || out->device() != x_.device() ||
              out->stride(-1) != 1))
    bad_value(what, ": out must be ", at::IntArrayRef(sizes), " in x's dtype with unit element stride");
  if (xm && (!g || g->scalar_type() != at::kFloat || xm->scalar_type() != at::kFloat || !g->is_contiguous() || !xm->is_contiguous() ||
             g->dim() != 2 || g->size(0) != M || xm->numel() != M || g->device() != x_.device() || xm->device() != x_.device()))
    bad_value(what, ": xm needs fp32 contiguous g [M, H] and xm [M] on x's device");
  no_grad(what, {&x_, &ws});
  for (const OptTensor* t : {&out, &xm, &g})
    if (*t) no_grad(what, {&**t});
  TORCH_CHECK(M <= INT_MAX && N <= INT_MAX && K <= INT_MAX, "int8_linear: sizes beyond 32 bits");
  const Tensor x = unit(x_.dim() == 2 ? x_ : x_.reshape({M, K}));
  Tensor y2;
  if (out) {
    y2 = out->dim() == 2 ? *out : out->view({M, N});  // an output that is no [M, N] in memory is refused
    if (M > 1 && y2.stride(0) < N) bad_value(what, ": the rows of out overlap");
    apart(y2, N, x, K, M, what);
  }
  on_gpu(x_, what);
  const On on(x_);
  const Tensor y = out ? *out : empty(sizes, x_, x_.scalar_type());
  if (!out) y2 = y.dim() == 2 ? y : y.view({M, N});
  a.M = int(M); a.N = int(N); a.K = int(K);
  a.x = x.data_ptr(); a.x_sr = x.stride(0);
  a.wq = static_cast<const int8_t*>(wq.data_ptr()); a.w_scale = fptr(ws);
  a.y = y2.data_ptr(); a.y_sr = y2.stride(0);
  a.run = run ? static_cast<const unsigned char*>(run->data_ptr()) : nullptr;
  if (xm) {
    a.g = fptr(*g); a.xm = fptr(*xm); a.heads = int(g->size(1));
  }
  Tensor wk;
  if (const size_t n = mote_int8_linear_workspace(&a)) {
    wk = bytes(n, x);
    a.workspace = wk.data_ptr();
    a.workspace_bytes = n;
  }
  check(mote_int8_linear(&a, on.stream), "mote_int8_linear");
  return y;
}

}  // namespace

PYBIND11_MODULE(_torch_launch, m) {
  // the interpreter lock is free while a call allocates and launches, as it was during the ctypes calls
  using nogil = py::call_guard<py::gil_scoped_release>;
  m.def("relation_fwd", &relation_fwd, nogil());
  m.def("relation_bwd", &relation_bwd, nogil());
  m.def("rope_givens", &rope_givens, nogil());
  m.def("rope_givens_bwd", &rope_givens_bwd, nogil());
  m.def("linear_wgrad", &linear_wgrad, nogil());
  m.def("add_rms_norm", &add_rms_norm, nogil());
  m.def("add_rms_norm_bwd", &add_rms_norm_bwd, nogil());
  m.def("qkv_rope", &qkv_rope, nogil());
  m.def("chunk_route", &chunk_route, nogil());
  m.def("dechunk", &dechunk, nogil());
  m.def("dechunk_bwd", &dechunk_bwd, nogil());
  m.def("cache4_write", &cache4_write, nogil());
  m.def("cache4_read", &cache4_read, nogil());
  m.def("relation_decode4", &relation_decode4, nogil());
  m.def("quantize_rows", &quantize_rows, nogil());
  m.def("int8_linear", &int8_linear, nogil());
}
