// torch operators over the C-ABI: a whole quantized linear (and a set of sibling linears) per call.
//
// svdq::linear and svdq::linear_siblings enqueue the activation pass and the GEMM back to back on the
// current stream, with every intermediate (operand codes, scales, low-rank activations, x_hat) in one
// workspace from the caching allocator.  As two Python operators with five allocations a layer call
// took 75 us on the host, three times a prompt-sized layer's GPU time; as one native operator 21 us
// (four sibling layers 172 -> 42 us).
// Registered with the dispatcher like any operator: tracing, vmap, dispatch modes and autograd meet
// them there (no gradient is defined).  The shape functions are registered from Python (ops.py).
#include <ATen/ATen.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/autograd_not_implemented_fallback.h>
#include <torch/library.h>

#include "../../include/svdq_gfx950.h"

namespace {

using at::Tensor;
using OptTensor = std::optional<Tensor>;

const char* status_name(int s) {
  switch (s) {
    case SVDQ_ERR_ARG: return "SVDQ_ERR_ARG";
    case SVDQ_ERR_SHAPE: return "SVDQ_ERR_SHAPE";
    case SVDQ_ERR_ALIGN: return "SVDQ_ERR_ALIGN";
    case SVDQ_ERR_UNSUPPORTED: return "SVDQ_ERR_UNSUPPORTED";
    case SVDQ_ERR_LAUNCH: return "SVDQ_ERR_LAUNCH";
  }
  return "SVDQ_ERR";
}
void check_status(const char* fn, int status) {
  TORCH_CHECK(status == SVDQ_OK, fn, " failed with ", status_name(status), ": ", svdq_last_error());
}

void check_tensor(const char* name, const Tensor& t, c10::Device dev, at::ScalarType dtype) {
  TORCH_CHECK_VALUE(t.device() == dev, name, " is on ", t.device(), ", expected ", dev);
  TORCH_CHECK_TYPE(t.scalar_type() == dtype, name, " must be ", dtype, ", got ", t.scalar_type());
  TORCH_CHECK_VALUE(t.is_contiguous(), name, " must be contiguous");
}

template <class T = void>
T* ptr(const Tensor& t) {
  return static_cast<T*>(t.data_ptr());
}
template <class T = void>
T* ptr(const OptTensor& t) {
  return t.has_value() ? static_cast<T*>(t->data_ptr()) : nullptr;
}

// One layer's operands, checked, and where its intermediates go in the workspace.
struct Layer {
  const Tensor *srs, *l2, *w, *ws, *l1cat;
  OptTensor lora_down, lora_mult, bias;
  int64_t rtp, n, r, rl;
  int splits;
  int64_t qa, sx, xhat, mid;   // byte offsets, -1: not used
};

constexpr int64_t kNone = -1;   // operand: x_hat only, the W4A16 path
bool fast_group(int64_t g) { return g == 64 || g == 128; }

int64_t operand_bytes(int64_t rows, int64_t k, int64_t operand) {
  return operand == SVDQ_OPERAND_E3M2 ? ((rows + 1) & ~int64_t(1)) * k * 3 / 4 : rows * k;
}

struct Call {
  c10::Device dev;
  int64_t m, k, group, operand, bytes = 0;
  bool quant, want_xhat;
  std::vector<int64_t> lead;
  Tensor x;

  // x [..., K'] with K' <= K: flattened to contiguous rows, zero columns up to K
  Call(const Tensor& xin, int64_t k_, int64_t group_, int64_t operand_)
      : dev(xin.device()), k(k_), group(group_), operand(operand_) {
    TORCH_CHECK(xin.is_cuda(), "svdq::linear needs a GPU tensor");
    TORCH_CHECK_TYPE(xin.scalar_type() == at::kBFloat16, "x must be bfloat16, got ", xin.scalar_type());
    TORCH_CHECK_VALUE(xin.dim() >= 2, "expected [..., K] activation, got shape ", xin.sizes());
    TORCH_CHECK_VALUE(group > 0 && k > 0 && k % group == 0, "K=", k, " must be a multiple of group_size=", group);
    TORCH_CHECK_VALUE(operand == kNone || operand == SVDQ_OPERAND_E4M3 || operand == SVDQ_OPERAND_I8 ||
                          operand == SVDQ_OPERAND_E3M2,
                      "operand=", operand);
    const int64_t kx = xin.size(-1);
    TORCH_CHECK_VALUE(kx <= k, "activation K=", kx, " exceeds packed weight K=", k);
    lead = xin.sizes().vec();
    lead.pop_back();
    m = 1;
    for (int64_t d : lead) m *= d;
    TORCH_CHECK_VALUE(m <= INT32_MAX && k <= INT32_MAX, "M=", m, ", K=", k, " exceed 2^31 - 1");
    x = xin.reshape({m, kx}).contiguous();
    if (kx != k) x = at::constant_pad_nd(x, {0, k - kx}, 0);
    quant = operand != kNone;
    want_xhat = !quant || !fast_group(group);
  }

  int64_t take(int64_t n) {
    const int64_t at = bytes;
    bytes += (n + 255) / 256 * 256;
    return at;
  }

  Layer layer(const Tensor& srs, const Tensor& l2, OptTensor lora_down, OptTensor lora_mult, int64_t rtp,
              const Tensor& w, const Tensor& ws, const Tensor& l1cat, OptTensor bias) {
    Layer l{&srs, &l2, &w, &ws, &l1cat, std::move(lora_down), std::move(lora_mult), std::move(bias)};
    l.rtp = rtp;
    check_tensor("srs", srs, dev, at::kFloat);
    TORCH_CHECK_VALUE(srs.numel() == 2 * k, "srs has ", srs.numel(), " elements, expected ", 2 * k);
    check_tensor("l2", l2, dev, at::kBFloat16);
    TORCH_CHECK_VALUE(l2.dim() == 2 && l2.size(1) == k, "l2 must be [r, ", k, "], got ", l2.sizes());
    l.r = l2.size(0);
    l.rl = 0;
    if (l.lora_down.has_value()) {
      check_tensor("lora_down", *l.lora_down, dev, at::kBFloat16);
      TORCH_CHECK_VALUE(l.lora_down->dim() == 2 && l.lora_down->size(1) == k, "lora_down must be [rl, ", k, "], got ",
                        l.lora_down->sizes());
      l.rl = l.lora_down->size(0);
      TORCH_CHECK_VALUE(l.lora_mult.has_value() && l.lora_mult->numel() == l.rl, "lora_mult must have rl entries");
      check_tensor("lora_mult", *l.lora_mult, dev, at::kFloat);
    }
    check_tensor("weight", w, dev, at::kByte);
    check_tensor("weight scales", ws, dev, quant ? at::kInt : at::kHalf);
    TORCH_CHECK_VALUE(ws.dim() == 2 && ws.size(quant ? 0 : 1) == k / group, "weight scales do not match K=", k,
                      ", group_size=", group, ": ", ws.sizes());
    l.n = ws.size(quant ? 1 : 0);
    TORCH_CHECK_VALUE(l.n <= INT32_MAX, "N=", l.n, " exceeds 2^31 - 1");
    TORCH_CHECK_VALUE(w.numel() == (quant ? operand_bytes(l.n, k, operand) : l.n * k / 2), "weight holds ", w.numel(),
                      " bytes for N=", l.n, ", K=", k);
    check_tensor("l1cat", l1cat, dev, at::kBFloat16);
    TORCH_CHECK_VALUE(l1cat.dim() == 2 && l1cat.size(0) == l.n && l1cat.size(1) == rtp, "l1cat must be [", l.n, ", ",
                      rtp, "], got ", l1cat.sizes());
    if (l.bias.has_value()) {
      check_tensor("bias", *l.bias, dev, at::kBFloat16);
      TORCH_CHECK_VALUE(l.bias->numel() == l.n, "bias must have ", l.n, " entries");
    }
    int64_t mid_floats = 0;
    check_status("svdq_act_quant_workspace",
                 svdq_act_quant_workspace((int)m, (int)k, (int)group, (int)rtp, &l.splits, &mid_floats));
    l.qa = quant ? take(operand_bytes(m, k, operand)) : -1;
    l.sx = quant ? take(4 * m * (k / group)) : -1;
    l.xhat = want_xhat ? take(2 * m * k) : -1;
    l.mid = take(4 * mid_floats);
    return l;
  }

  unsigned flags(bool exact) const {
    return (operand == SVDQ_OPERAND_E4M3 ? SVDQ_ACT_OPERAND_E4M3 : 0u) |
           (operand == SVDQ_OPERAND_I8 ? SVDQ_ACT_OPERAND_I8 : 0u) |
           (operand == SVDQ_OPERAND_E3M2 ? SVDQ_ACT_OPERAND_E3M2 : 0u) | (want_xhat ? SVDQ_ACT_XHAT : 0u) |
           (exact ? SVDQ_ACT_EXACT_DIV : 0u) | (quant ? SVDQ_ACT_SX_PAIRS : 0u);
  }

  void act_quant(const Layer& l, uint8_t* base, bool exact, hipStream_t st) const {
    auto at = [&](int64_t off) -> void* { return off < 0 ? nullptr : base + off; };
    check_status("svdq_act_quant",
                 svdq_act_quant(ptr(x), k, ptr<float>(*l.srs), ptr(*l.l2), (int)l.r, ptr(l.lora_down), (int)l.rl,
                                ptr<float>(l.lora_mult), (int)m, (int)k, (int)group, (int)l.rtp, flags(exact),
                                at(l.qa), at(l.sx), nullptr, at(l.xhat), k, static_cast<float*>(at(l.mid)), l.splits,
                                st));
  }

  Tensor output(const Layer& l, bool out_f32) const {
    std::vector<int64_t> shape = lead;
    shape.push_back(l.n);
    return at::empty(shape, x.options().dtype(out_f32 ? at::kFloat : at::kBFloat16));
  }
};

Tensor linear(const Tensor& x, const Tensor& srs, const Tensor& l2, const OptTensor& lora_down,
              const OptTensor& lora_mult, int64_t group, int64_t rtp, const Tensor& weight, const Tensor& weight_scales,
              const Tensor& l1cat, const OptTensor& bias, int64_t operand, bool out_f32, bool exact, int64_t epi,
              const OptTensor& aux, const OptTensor& vec) {
  TORCH_CHECK_VALUE(srs.numel() % 2 == 0, "srs must hold 2 K values");
  Call c(x, srs.numel() / 2, group, operand);
  const c10::DeviceGuard guard(c.dev);
  const Layer l = c.layer(srs, l2, lora_down, lora_mult, rtp, weight, weight_scales, l1cat, bias);
  if (epi != SVDQ_EPI_NONE) {
    TORCH_CHECK_VALUE(!out_f32, "epilogue ops need bf16 output");
    TORCH_CHECK_VALUE(aux.has_value(), "epilogue op needs aux");
    check_tensor("aux", *aux, c.dev, at::kBFloat16);
    TORCH_CHECK_VALUE(aux->numel() == c.m * l.n, "aux must be [", c.m, ", ", l.n, "], got ", aux->sizes());
    TORCH_CHECK_VALUE(vec.has_value() == (epi == SVDQ_EPI_RESIDUAL_GATE), "vec is for residual_gate");
    if (vec.has_value()) {
      check_tensor("vec", *vec, c.dev, at::kBFloat16);
      TORCH_CHECK_VALUE(vec->numel() == l.n, "vec must have ", l.n, " entries");
    }
  } else {
    TORCH_CHECK_VALUE(!aux.has_value() && !vec.has_value(), "aux / vec given without an epilogue op");
  }
  Tensor y = c.output(l, out_f32);
  const Tensor work = at::empty({c.bytes}, c.x.options().dtype(at::kByte));
  uint8_t* base = ptr<uint8_t>(work);
  const hipStream_t st = c10::hip::getCurrentHIPStream(c.dev.index());
  c.act_quant(l, base, exact, st);
  const int m = (int)c.m, n = (int)l.n, k = (int)c.k, rt = (int)rtp, f32 = out_f32;
  if (c.quant)
    check_status("svdq_w4a4_gemm_epi",
                 svdq_w4a4_gemm_epi(base + l.qa, (int)operand, base + l.sx, ptr(weight), ptr(weight_scales),
                                    base + l.mid, ptr(l1cat), rt, ptr(bias), m, n, k, (int)group, ptr(y), n, f32,
                                    (int)epi, ptr(aux), n, ptr(vec), st));
  else
    check_status("svdq_w4a16_gemm_epi",
                 svdq_w4a16_gemm_epi(base + l.xhat, k, ptr(weight), ptr(weight_scales), base + l.mid, ptr(l1cat), rt,
                                     ptr(bias), m, n, k, (int)group, ptr(y), n, f32, (int)epi, ptr(aux), n, ptr(vec),
                                     st));
  return y;
}

std::vector<Tensor> linear_siblings(const Tensor& x, const std::vector<Tensor>& srs, const std::vector<Tensor>& l2,
                                    const c10::List<OptTensor>& lora_down, const c10::List<OptTensor>& lora_mult,
                                    int64_t group, c10::IntArrayRef rtp, const std::vector<Tensor>& weight,
                                    const std::vector<Tensor>& weight_scales, const std::vector<Tensor>& l1cat,
                                    const c10::List<OptTensor>& bias, int64_t operand, bool out_f32, bool exact) {
  const size_t count = srs.size();
  TORCH_CHECK_VALUE(count >= 1 && count <= SVDQ_MAX_SIBLINGS, "1..", SVDQ_MAX_SIBLINGS, " sibling layers, got ", count);
  TORCH_CHECK_VALUE(l2.size() == count && lora_down.size() == count && lora_mult.size() == count &&
                        rtp.size() == count && weight.size() == count && weight_scales.size() == count &&
                        l1cat.size() == count && bias.size() == count,
                    "one entry per layer in every list");
  TORCH_CHECK_VALUE(srs[0].numel() % 2 == 0, "srs must hold 2 K values");
  Call c(x, srs[0].numel() / 2, group, operand);
  TORCH_CHECK_VALUE(fast_group(group), "sibling launch needs group size 64 or 128, got ", group);
  const c10::DeviceGuard guard(c.dev);
  Layer l[SVDQ_MAX_SIBLINGS];
  std::vector<Tensor> ys;
  bool one_pass = operand == SVDQ_OPERAND_E3M2 || !c.quant;   // one launch for the activation passes
  for (size_t i = 0; i < count; ++i) {
    l[i] = c.layer(srs[i], l2[i], lora_down.get(i), lora_mult.get(i), rtp[i], weight[i], weight_scales[i], l1cat[i],
                   bias.get(i));
    ys.push_back(c.output(l[i], out_f32));
    one_pass = one_pass && !l[i].rl && rtp[i] == rtp[0];
  }
  const Tensor work = at::empty({c.bytes}, c.x.options().dtype(at::kByte));
  uint8_t* base = ptr<uint8_t>(work);
  const hipStream_t st = c10::hip::getCurrentHIPStream(c.dev.index());
  const int m = (int)c.m, k = (int)c.k, f32 = out_f32;
  if (one_pass) {
    svdq_act_sibling a[SVDQ_MAX_SIBLINGS];
    for (size_t i = 0; i < count; ++i)
      a[i] = {ptr<float>(srs[i]), ptr(l2[i]), (int)l[i].r, base + (c.quant ? l[i].qa : l[i].xhat),
              c.quant ? base + l[i].sx : nullptr, reinterpret_cast<float*>(base + l[i].mid)};
    if (c.quant)
      check_status("svdq_act_quant_siblings", svdq_act_quant_siblings(ptr(c.x), k, a, (int)count, m, k, (int)group,
                                                                      (int)rtp[0], c.flags(exact), l[0].splits, st));
    else
      check_status("svdq_act_xhat_siblings", svdq_act_xhat_siblings(ptr(c.x), k, a, (int)count, m, k, (int)group,
                                                                    (int)rtp[0], exact, l[0].splits, st));
  } else {
    for (size_t i = 0; i < count; ++i) c.act_quant(l[i], base, exact, st);
  }
  if (c.quant) {
    svdq_w4a4_sibling g[SVDQ_MAX_SIBLINGS];
    for (size_t i = 0; i < count; ++i)
      g[i] = {base + l[i].qa, base + l[i].sx, ptr(weight[i]), ptr(weight_scales[i]), base + l[i].mid, ptr(l1cat[i]),
              (int)rtp[i], ptr(l[i].bias), (int)l[i].n, ptr(ys[i]), l[i].n};
    check_status("svdq_w4a4_gemm_siblings",
                 svdq_w4a4_gemm_siblings(g, (int)count, (int)operand, m, k, (int)group, f32, st));
  } else {
    svdq_w4a16_sibling g[SVDQ_MAX_SIBLINGS];
    for (size_t i = 0; i < count; ++i)
      g[i] = {base + l[i].xhat, k, ptr(weight[i]), ptr(weight_scales[i]), base + l[i].mid, ptr(l1cat[i]), (int)rtp[i],
              ptr(l[i].bias), (int)l[i].n, ptr(ys[i]), l[i].n};
    check_status("svdq_w4a16_gemm_siblings", svdq_w4a16_gemm_siblings(g, (int)count, m, k, (int)group, f32, st));
  }
  return ys;
}

// ---- Microscaled blocks --------------------------------------------------------------------------
// Codes are uint8 [..., kp / 2] (E2M1) or float8_e4m3fn [..., kp] (E4M3), scales float8_e8m0fnu [..., sp] (taken as uint8
// bytes too), with kp and sp as in svdq_gfx950.h.  Native operators like the linears: a prompt-sized call is shorter on the
// GPU than a Python operator's checks and allocations.

int64_t mx_kp(int64_t k) { return (k + 127) / 128 * 128; }
int64_t mx_sp(int64_t k) { return (k + 511) / 512 * 16; }
int64_t mx_row_bytes(int64_t k, int64_t fmt) { return fmt == SVDQ_MX_E4M3 ? mx_kp(k) : mx_kp(k) / 2; }

void check_fmt(int64_t fmt) {
  TORCH_CHECK_VALUE(fmt == SVDQ_MX_E2M1 || fmt == SVDQ_MX_E4M3, "fmt=", fmt);
}

// [..., K] as rows: the last dimension dense, the leading ones flattened (a copy where they have no common stride)
struct Rows {
  Tensor t;
  int64_t m, k, ld;
  std::vector<int64_t> lead;

  // aligned: 16-byte rows, copied where they are not
  Rows(const char* name, const Tensor& x, bool aligned = false) {
    TORCH_CHECK_TYPE(x.scalar_type() == at::kBFloat16, name, " must be bfloat16, got ", x.scalar_type());
    TORCH_CHECK_VALUE(x.dim() >= 1 && x.size(-1) > 0, name, " must be [..., K] with K > 0, got ", x.sizes());
    lead = x.sizes().vec();
    k = lead.back();
    lead.pop_back();
    m = 1;
    for (int64_t d : lead) m *= d;
    TORCH_CHECK_VALUE(m <= INT32_MAX && k <= 1 << 30, name, ": ", m, " rows of ", k, " columns are too many");
    t = x.dim() == 2 ? x : x.reshape({m, k});
    if (t.stride(1) != 1 && k > 1) t = t.contiguous();
    ld = m > 1 ? t.stride(0) : k;
    if (ld < k || (aligned && (ld % 8 || reinterpret_cast<uintptr_t>(t.data_ptr()) % 16))) {
      t = at::empty({m, k}, t.options()).copy_(t);
      ld = k;
    }
  }
};

// new codes and scales of the rows of x
std::tuple<Tensor, Tensor> mx_empty(const Rows& r, int64_t fmt) {
  std::vector<int64_t> cs = r.lead, ss = r.lead;
  cs.push_back(mx_row_bytes(r.k, fmt));
  ss.push_back(mx_sp(r.k));
  return {at::empty(cs, r.t.options().dtype(fmt == SVDQ_MX_E4M3 ? at::kFloat8_e4m3fn : at::kByte)),
          at::empty(ss, r.t.options().dtype(at::kFloat8_e8m0fnu))};
}

// codes and their scales, checked: format, rows and padded columns
struct Mx {
  int64_t fmt, m, kp;
  std::vector<int64_t> lead;

  Mx(const char* name, const Tensor& codes, const Tensor& scales, c10::Device dev) {
    const auto dt = codes.scalar_type();
    TORCH_CHECK_TYPE(dt == at::kByte || dt == at::kFloat8_e4m3fn, name, " must be uint8 (E2M1) or float8_e4m3fn codes, got ", dt);
    check_tensor(name, codes, dev, dt);
    check_tensor("their scales", scales, dev, scales.scalar_type() == at::kByte ? at::kByte : at::kFloat8_e8m0fnu);
    fmt = dt == at::kByte ? SVDQ_MX_E2M1 : SVDQ_MX_E4M3;
    TORCH_CHECK_VALUE(codes.dim() >= 1, name, " must be [..., K], got ", codes.sizes());
    lead = codes.sizes().vec();
    kp = lead.back() * (fmt == SVDQ_MX_E2M1 ? 2 : 1);
    lead.pop_back();
    m = 1;
    for (int64_t d : lead) m *= d;
    TORCH_CHECK_VALUE(kp > 0 && kp % 128 == 0 && kp <= 1 << 30 && m <= INT32_MAX, name,
                      " must hold rows of a multiple of 128 values, got ", codes.sizes());
    std::vector<int64_t> want = lead;
    want.push_back(mx_sp(kp));
    TORCH_CHECK_VALUE(scales.sizes() == at::IntArrayRef(want), name, "' scales must be ", at::IntArrayRef(want), ", got ",
                      scales.sizes());
  }
};

hipStream_t stream_of(c10::Device dev) { return c10::hip::getCurrentHIPStream(dev.index()); }

std::tuple<Tensor, Tensor> mx_quantize(const Tensor& x, int64_t fmt) {
  check_fmt(fmt);
  const c10::DeviceGuard guard(x.device());
  const Rows r("x", x);
  auto [codes, scales] = mx_empty(r, fmt);
  check_status("svdq_mx_quantize", svdq_mx_quantize(ptr(r.t), r.ld, (int)r.m, (int)r.k, (int)fmt, ptr(codes), ptr(scales),
                                                    stream_of(x.device())));
  return {codes, scales};
}

Tensor mx_dequantize(const Tensor& codes, const Tensor& scales, int64_t k) {
  const c10::DeviceGuard guard(codes.device());
  const Mx a("codes", codes, scales, codes.device());
  TORCH_CHECK_VALUE(k > 0 && mx_kp(k) == a.kp, "k=", k, " does not pad to the codes' ", a.kp, " columns");
  std::vector<int64_t> shape = a.lead;
  shape.push_back(k);
  Tensor y = at::empty(shape, codes.options().dtype(at::kBFloat16));
  check_status("svdq_mx_dequantize", svdq_mx_dequantize(ptr(codes), ptr(scales), (int)a.m, (int)k, (int)a.fmt, ptr(y),
                                                        stream_of(codes.device())));
  return y;
}

// y [lead..., N] = a w^T + bias of checked activation blocks (codes at a, scales at as)
Tensor mx_product(const void* a, const void* as, int64_t fmt, int64_t m, int64_t kp, std::vector<int64_t> lead,
                  const Tensor& w, const Tensor& w_scales, const OptTensor& bias, bool out_f32) {
  const c10::Device dev = w.device();
  const Mx b("w", w, w_scales, dev);
  TORCH_CHECK_TYPE(b.fmt == SVDQ_MX_E2M1, "w must be uint8 (E2M1) codes");
  TORCH_CHECK_VALUE(w.dim() == 2 && b.m > 0, "w must be [N, K / 2] codes, got ", w.sizes());
  TORCH_CHECK_VALUE(b.kp == kp, "rows of ", kp, " values (padded) against a weight of ", b.kp);
  if (bias.has_value()) {
    check_tensor("bias", *bias, dev, at::kBFloat16);
    TORCH_CHECK_VALUE(bias->numel() == b.m, "bias must have ", b.m, " entries, got ", bias->numel());
  }
  lead.push_back(b.m);
  Tensor y = at::empty(lead, w.options().dtype(out_f32 ? at::kFloat : at::kBFloat16));
  check_status("svdq_mx_gemm", svdq_mx_gemm(a, as, (int)fmt, ptr(w), ptr(w_scales), ptr(bias), (int)m, (int)b.m, (int)kp,
                                            ptr(y), b.m, out_f32, stream_of(dev)));
  return y;
}

Tensor mx_gemm(const Tensor& a, const Tensor& a_scales, const Tensor& w, const Tensor& w_scales, const OptTensor& bias,
               bool out_f32) {
  const c10::DeviceGuard guard(w.device());
  const Mx r("a", a, a_scales, w.device());
  return mx_product(ptr(a), ptr(a_scales), r.fmt, r.m, r.kp, r.lead, w, w_scales, bias, out_f32);
}

Tensor mx_linear(const Tensor& x, const Tensor& w, const Tensor& w_scales, const OptTensor& bias, int64_t fmt,
                 bool out_f32) {
  check_fmt(fmt);
  const c10::DeviceGuard guard(w.device());
  TORCH_CHECK_VALUE(x.device() == w.device(), "x is on ", x.device(), ", expected ", w.device());
  const Rows r("x", x);
  const int64_t codes = r.m * mx_row_bytes(r.k, fmt);   // rows of 64 bytes and more: 16-byte aligned scales behind
  const Tensor work = at::empty({codes + r.m * mx_sp(r.k)}, r.t.options().dtype(at::kByte));
  uint8_t* base = ptr<uint8_t>(work);
  check_status("svdq_mx_quantize", svdq_mx_quantize(ptr(r.t), r.ld, (int)r.m, (int)r.k, (int)fmt, base, base + codes,
                                                    stream_of(w.device())));
  return mx_product(base, base + codes, fmt, r.m, mx_kp(r.k), r.lead, w, w_scales, bias, out_f32);
}

std::tuple<Tensor, Tensor> silu_mul_mx(const Tensor& gate, const Tensor& up, int64_t fmt) {
  check_fmt(fmt);
  const c10::DeviceGuard guard(gate.device());
  TORCH_CHECK_VALUE(up.device() == gate.device(), "up is on ", up.device(), ", expected ", gate.device());
  TORCH_CHECK_VALUE(up.sizes() == gate.sizes(), "gate ", gate.sizes(), " and up ", up.sizes(), " differ");
  const Rows g("gate", gate), u("up", up);
  auto [codes, scales] = mx_empty(g, fmt);
  check_status("svdq_silu_mul_mx", svdq_silu_mul_mx(ptr(g.t), g.ld, ptr(u.t), u.ld, (int)g.m, (int)g.k, (int)fmt,
                                                    ptr(codes), ptr(scales), stream_of(gate.device())));
  return {codes, scales};
}

// a vector [H] of the norms, 16-byte aligned
Tensor norm_vector(const char* name, const Tensor& t, int64_t h, c10::Device dev) {
  check_tensor(name, t, dev, at::kBFloat16);
  TORCH_CHECK_VALUE(t.numel() == h, name, " must have ", h, " elements, got ", t.numel());
  return reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 ? t.clone() : t;
}

std::tuple<Tensor, Tensor> rms_norm_modulate_mx(const Tensor& x, const Tensor& weight, const Tensor& shift, double eps,
                                                int64_t fmt) {
  check_fmt(fmt);
  const c10::DeviceGuard guard(x.device());
  const Rows r("x", x, true);
  TORCH_CHECK_VALUE(r.k % 8 == 0, "rows must be multiples of 8 values, got ", r.k);
  const Tensor w = norm_vector("weight", weight, r.k, x.device()), s = norm_vector("shift", shift, r.k, x.device());
  auto [codes, scales] = mx_empty(r, fmt);
  check_status("svdq_rms_norm_modulate_mx",
               svdq_rms_norm_modulate_mx(ptr(r.t), r.ld, ptr(w), ptr(s), (int)r.m, (int)r.k, (float)eps, (int)fmt,
                                         ptr(codes), ptr(scales), stream_of(x.device())));
  return {codes, scales};
}

std::tuple<Tensor, Tensor, Tensor> residual_rms_norm_modulate_mx(const Tensor& x, const Tensor& v, const Tensor& gate,
                                                                 const Tensor& weight, const Tensor& shift, double eps,
                                                                 int64_t fmt) {
  check_fmt(fmt);
  const c10::DeviceGuard guard(x.device());
  TORCH_CHECK_VALUE(v.device() == x.device(), "v is on ", v.device(), ", expected ", x.device());
  TORCH_CHECK_VALUE(v.sizes() == x.sizes(), "v ", v.sizes(), " must match x ", x.sizes());
  const Rows r("x", x, true), rv("v", v, true);
  TORCH_CHECK_VALUE(r.k % 8 == 0, "rows must be multiples of 8 values, got ", r.k);
  const Tensor g = norm_vector("gate", gate, r.k, x.device()), w = norm_vector("weight", weight, r.k, x.device()),
               s = norm_vector("shift", shift, r.k, x.device());
  Tensor xo = at::empty(x.sizes(), r.t.options());
  auto [codes, scales] = mx_empty(r, fmt);
  check_status("svdq_residual_rms_norm_modulate_mx",
               svdq_residual_rms_norm_modulate_mx(ptr(r.t), r.ld, ptr(rv.t), rv.ld, ptr(g), ptr(w), ptr(s), (int)r.m,
                                                  (int)r.k, (float)eps, (int)fmt, ptr(xo), r.k, ptr(codes), ptr(scales),
                                                  stream_of(x.device())));
  return {xo, codes, scales};
}

// ---- 8-bit floating point with a scale per block ---------------------------------------------------
// Codes are float8_e4m3fn [..., kp], scales float32: an activation's [kp / 128, rows], a weight's [ceil(N / 128), kp / 128].

std::tuple<Tensor, Tensor> fp8_quantize(const Tensor& x) {
  const c10::DeviceGuard guard(x.device());
  const Rows r("x", x);
  std::vector<int64_t> cs = r.lead;
  cs.push_back(mx_kp(r.k));
  Tensor codes = at::empty(cs, r.t.options().dtype(at::kFloat8_e4m3fn));
  Tensor scales = at::empty({mx_kp(r.k) / 128, r.m}, r.t.options().dtype(at::kFloat));
  check_status("svdq_fp8_quantize", svdq_fp8_quantize(ptr(r.t), r.ld, (int)r.m, (int)r.k, ptr(codes), ptr<float>(scales),
                                                      stream_of(x.device())));
  return {codes, scales};
}

// w, w_scales and bias for rows of kp codes; y [lead..., N]
Tensor fp8_output(int64_t kp, std::vector<int64_t> lead, const Tensor& w, const Tensor& w_scales, const OptTensor& bias) {
  const c10::Device dev = w.device();
  check_tensor("w", w, dev, at::kFloat8_e4m3fn);
  TORCH_CHECK_VALUE(w.dim() == 2 && w.size(0) > 0 && w.size(0) <= INT32_MAX, "w must be [N, K] codes, got ", w.sizes());
  TORCH_CHECK_VALUE(w.size(1) == kp, "rows of ", kp, " values (padded to 128) against a weight of ", w.size(1));
  const int64_t n = w.size(0);
  check_tensor("w_scales", w_scales, dev, at::kFloat);
  const std::vector<int64_t> want{(n + 127) / 128, kp / 128};
  TORCH_CHECK_VALUE(w_scales.sizes() == at::IntArrayRef(want), "w_scales must be ", at::IntArrayRef(want), ", got ",
                    w_scales.sizes());
  if (bias.has_value()) {
    check_tensor("bias", *bias, dev, at::kBFloat16);
    TORCH_CHECK_VALUE(bias->numel() == n, "bias must have ", n, " entries, got ", bias->numel());
  }
  lead.push_back(n);
  return at::empty(lead, w.options().dtype(at::kBFloat16));
}

Tensor fp8_gemm(const Tensor& a, const Tensor& a_scales, const Tensor& w, const Tensor& w_scales, const OptTensor& bias) {
  const c10::Device dev = w.device();
  const c10::DeviceGuard guard(dev);
  check_tensor("a", a, dev, at::kFloat8_e4m3fn);
  TORCH_CHECK_VALUE(a.dim() >= 1 && a.size(-1) > 0 && a.size(-1) % 128 == 0 && a.size(-1) <= 1 << 30, "a must be [..., K] "
                    "codes, K a multiple of 128, got ", a.sizes());
  std::vector<int64_t> lead = a.sizes().vec();
  const int64_t kp = lead.back(), m = a.numel() / kp;
  lead.pop_back();
  TORCH_CHECK_VALUE(m <= INT32_MAX, "a: ", m, " rows are too many");
  check_tensor("a_scales", a_scales, dev, at::kFloat);
  const std::vector<int64_t> want{kp / 128, m};
  TORCH_CHECK_VALUE(a_scales.sizes() == at::IntArrayRef(want), "a_scales must be ", at::IntArrayRef(want), ", got ",
                    a_scales.sizes());
  const Tensor y = fp8_output(kp, lead, w, w_scales, bias);
  check_status("svdq_fp8_gemm", svdq_fp8_gemm(ptr(a), ptr<float>(a_scales), ptr(w), ptr<float>(w_scales), ptr(bias), (int)m,
                                              (int)w.size(0), (int)kp, ptr(y), w.size(0), stream_of(dev)));
  return y;
}

Tensor fp8_linear(const Tensor& x, const Tensor& w, const Tensor& w_scales, const OptTensor& bias) {
  const c10::Device dev = w.device();
  const c10::DeviceGuard guard(dev);
  TORCH_CHECK_VALUE(x.device() == dev, "x is on ", x.device(), ", expected ", dev);
  const Rows r("x", x);
  const Tensor y = fp8_output(mx_kp(r.k), r.lead, w, w_scales, bias);
  const int n = (int)w.size(0);
  const Tensor work = at::empty({svdq_fp8_linear_workspace((int)r.m, (int)r.k)}, w.options().dtype(at::kByte));
  check_status("svdq_fp8_linear", svdq_fp8_linear(ptr(r.t), r.ld, ptr(w), ptr<float>(w_scales), ptr(bias), (int)r.m, n,
                                                  (int)r.k, ptr(y), n, ptr(work), stream_of(dev)));
  return y;
}

// [T, heads, D] with dense heads on 16 bytes; `packed`: heads one behind another
Tensor heads_of(const char* name, const Tensor& t, c10::Device dev, bool packed) {
  TORCH_CHECK_VALUE(t.device() == dev, name, " is on ", t.device(), ", expected ", dev);
  TORCH_CHECK_TYPE(t.scalar_type() == at::kBFloat16, name, " must be bfloat16, got ", t.scalar_type());
  TORCH_CHECK_VALUE(t.dim() == 3 && t.size(1) > 0 && t.size(0) <= INT32_MAX && t.size(1) <= INT32_MAX, name,
                    " must be [tokens, heads, dim], got ", t.sizes());
  const bool fits = t.stride(2) == 1 && (packed ? t.stride(1) == t.size(2) : t.stride(1) % 8 == 0 && t.stride(1) <= INT32_MAX) &&
                    t.stride(0) % 8 == 0 && reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0;
  return fits ? t : t.clone(at::MemoryFormat::Contiguous);
}

std::tuple<Tensor, Tensor> qk_norm_rope(const Tensor& q, const Tensor& k, const OptTensor& q_weight,
                                        const OptTensor& k_weight, const Tensor& cos, const Tensor& sin, double eps,
                                        const OptTensor& positions, bool interleaved) {
  const c10::Device dev = q.device();
  const c10::DeviceGuard guard(dev);
  const Tensor qh = heads_of("q", q, dev, false), kh = heads_of("k", k, dev, false);
  const int64_t t = q.size(0), d = q.size(2);
  TORCH_CHECK_VALUE(k.size(0) == t && k.size(2) == d, "k ", k.sizes(), " must have q's tokens and channels ", q.sizes());
  TORCH_CHECK_VALUE(d > 0 && d <= 256 && d % 16 == 0, "heads must have a multiple of 16 channels up to 256, got ", d);
  auto weight = [&](const char* name, const OptTensor& w) -> OptTensor {
    if (!w.has_value()) return w;
    return norm_vector(name, *w, d, dev);
  };
  const OptTensor qw = weight("q_weight", q_weight), kw = weight("k_weight", k_weight);
  const bool wide = cos.scalar_type() == at::kFloat;
  auto table = [&](const char* name, const Tensor& x) {
    TORCH_CHECK_VALUE(x.device() == dev, name, " is on ", x.device(), ", expected ", dev);
    TORCH_CHECK_TYPE(x.scalar_type() == (wide ? at::kFloat : at::kBFloat16), "cos and sin must both be float32 or bfloat16, got ",
                     cos.scalar_type(), " and ", sin.scalar_type());
    TORCH_CHECK_VALUE(x.dim() == 2 && x.size(0) > 0 && x.size(0) <= INT32_MAX && x.size(1) >= d / 2, name,
                      " must be [positions, >= ", d / 2, "], got ", x.sizes());
    const bool fits = x.stride(1) == 1 && x.stride(0) >= d / 2 && x.stride(0) * (wide ? 4 : 2) % 16 == 0 &&
                      reinterpret_cast<uintptr_t>(x.data_ptr()) % 16 == 0;
    return fits ? x : x.narrow(1, 0, d / 2).clone(at::MemoryFormat::Contiguous);
  };
  Tensor c = table("cos", cos), s = table("sin", sin);
  TORCH_CHECK_VALUE(c.size(0) == s.size(0), "cos ", cos.sizes(), " and sin ", sin.sizes(), " differ");
  if (c.stride(0) != s.stride(0)) {
    c = c.narrow(1, 0, d / 2).clone(at::MemoryFormat::Contiguous);
    s = s.narrow(1, 0, d / 2).clone(at::MemoryFormat::Contiguous);
  }
  OptTensor at_;
  if (positions.has_value()) {
    TORCH_CHECK_VALUE(positions->device() == dev, "positions are on ", positions->device(), ", expected ", dev);
    TORCH_CHECK_TYPE(positions->scalar_type() == at::kLong || positions->scalar_type() == at::kInt,
                     "positions must be int64 or int32, got ", positions->scalar_type());
    TORCH_CHECK_VALUE(positions->dim() == 1 && positions->size(0) == t, "positions must be [", t, "], got ", positions->sizes());
    at_ = positions->to(at::kLong).contiguous();
  } else {
    TORCH_CHECK_VALUE(c.size(0) >= t, "tables of ", c.size(0), " positions for ", t, " tokens");
  }
  Tensor qo = at::empty(q.sizes(), qh.options()), ko = at::empty(k.sizes(), kh.options());
  check_status("svdq_qk_norm_rope",
               svdq_qk_norm_rope(ptr(qh), qh.stride(0), (int)qh.stride(1), ptr(kh), kh.stride(0), (int)kh.stride(1), ptr(qw),
                                 ptr(kw), ptr(c), ptr(s), c.stride(0), (int)c.size(0), wide, ptr<int64_t>(at_), (int)t,
                                 (int)q.size(1), (int)k.size(1), (int)d, (float)eps, interleaved, ptr(qo), ptr(ko),
                                 stream_of(dev)));
  return {qo, ko};
}

// ---- The 8-bit cache of keys and values ---------------------------------------------------------------

struct Kv8 {
  int n, b, w, p, hkv, d;

  Kv8(int64_t tokens, const Tensor& offsets, const Tensor& lengths, const Tensor& table, const Tensor& k_codes,
      const Tensor& v_codes, const Tensor& scales, c10::Device dev) {
    check_tensor("k_codes", k_codes, dev, at::kFloat8_e4m3fn);
    check_tensor("v_codes", v_codes, dev, at::kFloat8_e4m3fn);
    check_tensor("scales", scales, dev, at::kFloat);
    check_tensor("cu_seqlens", offsets, dev, at::kInt);
    check_tensor("lengths", lengths, dev, at::kInt);
    check_tensor("block_table", table, dev, at::kInt);
    TORCH_CHECK_VALUE(k_codes.dim() == 4 && k_codes.size(2) == 64, "k_codes must be [pages, heads, 64, dim], got ", k_codes.sizes());
    const int64_t pages = k_codes.size(0), heads = k_codes.size(1), dim = k_codes.size(3);
    TORCH_CHECK_VALUE(dim == 64 || dim == 128, "heads must have 64 or 128 channels, got ", dim);
    const std::vector<int64_t> vs{pages, heads, dim, 64}, ss{pages, heads, 2};
    TORCH_CHECK_VALUE(v_codes.sizes() == at::IntArrayRef(vs), "v_codes must be ", at::IntArrayRef(vs), ", got ", v_codes.sizes());
    TORCH_CHECK_VALUE(scales.sizes() == at::IntArrayRef(ss), "scales must be ", at::IntArrayRef(ss), ", got ", scales.sizes());
    TORCH_CHECK_VALUE(table.dim() == 2, "block_table must be [sequences, pages], got ", table.sizes());
    const int64_t batch = table.size(0), width = table.size(1);
    TORCH_CHECK_VALUE(lengths.dim() == 1 && lengths.size(0) == batch && offsets.dim() == 1 && offsets.size(0) == batch + 1,
                      "lengths must be [", batch, "] and cu_seqlens [", batch + 1, "], got ", lengths.sizes(), " and ", offsets.sizes());
    TORCH_CHECK_VALUE(tokens <= INT32_MAX && pages > 0 && heads > 0 && batch > 0 && width > 0 && pages <= INT32_MAX &&
                      heads <= INT32_MAX && batch < INT32_MAX && width <= 1 << 24, "a cache of ", pages, " pages of ", heads,
                      " heads, a table of ", table.sizes(), ", ", tokens, " tokens");
    n = (int)tokens, b = (int)batch, w = (int)width, p = (int)pages, hkv = (int)heads, d = (int)dim;
  }
};

void kv8_append(const Tensor& k, const Tensor& v, const Tensor& cu_seqlens, const Tensor& lengths, const Tensor& block_table,
                const Tensor& k_codes, const Tensor& v_codes, const Tensor& scales) {
  const c10::Device dev = k_codes.device();
  const c10::DeviceGuard guard(dev);
  TORCH_CHECK(!(at::GradMode::is_enabled() && (k.requires_grad() || v.requires_grad())),
              "svdq::kv8_append has no gradient: its inputs may not require one");
  const Tensor kh = heads_of("k", k, dev, true), vh = heads_of("v", v, dev, true);
  const Kv8 c(k.size(0), cu_seqlens, lengths, block_table, k_codes, v_codes, scales, dev);
  TORCH_CHECK_VALUE(k.sizes() == v.sizes() && k.size(1) == c.hkv && k.size(2) == c.d, "k and v must be [tokens, ", c.hkv, ", ",
                    c.d, "], got ", k.sizes(), " and ", v.sizes());
  check_status("svdq_kv8_append",
               svdq_kv8_append(ptr(kh), kh.stride(0), ptr(vh), vh.stride(0), c.n, ptr<int>(cu_seqlens), ptr<int>(lengths),
                               ptr<int>(block_table), c.b, c.w, ptr(k_codes), ptr(v_codes), ptr<float>(scales), c.p, c.hkv,
                               c.d, stream_of(dev)));
  for (const Tensor* t : {&k_codes, &v_codes, &scales})
    if (!t->is_inference()) t->unsafeGetTensorImpl()->bump_version();
}

Tensor kv8_attention(const Tensor& q, const Tensor& cu_seqlens, const Tensor& lengths, const Tensor& block_table,
                     const Tensor& k_codes, const Tensor& v_codes, const Tensor& scales, double scale, bool causal) {
  const c10::Device dev = q.device();
  const c10::DeviceGuard guard(dev);
  const Tensor qh = heads_of("q", q, dev, true);
  const Kv8 c(q.size(0), cu_seqlens, lengths, block_table, k_codes, v_codes, scales, dev);
  TORCH_CHECK_VALUE(q.size(2) == c.d && q.size(1) % c.hkv == 0, "q must be [tokens, a multiple of ", c.hkv, ", ", c.d, "], got ",
                    q.sizes());
  const int h = (int)q.size(1);
  Tensor out = at::empty(q.sizes(), qh.options());
  const int64_t bytes = svdq_kv8_attention_workspace(c.n, c.b, c.w, h, c.hkv, c.d, causal);
  const Tensor work = bytes ? at::empty({bytes}, qh.options().dtype(at::kByte)) : Tensor();
  check_status("svdq_kv8_attention",
               svdq_kv8_attention(ptr(qh), qh.stride(0), c.n, ptr<int>(cu_seqlens), ptr<int>(lengths), ptr<int>(block_table),
                                  c.b, c.w, ptr(k_codes), ptr(v_codes), ptr<float>(scales), c.p, h, c.hkv, c.d, (float)scale,
                                  causal, ptr(out), bytes ? ptr(work) : nullptr, stream_of(dev)));
  return out;
}

}  // namespace

// The torch that this file was compiled against, found in the file by kernels/hip/lib.py ahead of
// loading it: the C++ interfaces used here hold for that build of torch only.
extern "C" __attribute__((used, visibility("default"))) const char svdq_torch_build[] = "svdq_torch built with torch " SVDQ_TORCH_BUILD;

TORCH_LIBRARY_FRAGMENT(svdq, m) {
  m.def(
      "linear(Tensor x, Tensor srs, Tensor l2, Tensor? lora_down, Tensor? lora_mult, int group_size, int rtp, "
      "Tensor weight, Tensor weight_scales, Tensor l1cat, Tensor? bias, int operand, bool out_f32, bool exact, "
      "int epi=0, Tensor? aux=None, Tensor? vec=None) -> Tensor");
  m.def(
      "linear_siblings(Tensor x, Tensor[] srs, Tensor[] l2, Tensor?[] lora_down, Tensor?[] lora_mult, "
      "int group_size, int[] rtp, Tensor[] weight, Tensor[] weight_scales, Tensor[] l1cat, Tensor?[] bias, "
      "int operand, bool out_f32, bool exact) -> Tensor[]");
  m.def("mx_quantize(Tensor x, int fmt) -> (Tensor, Tensor)");
  m.def("mx_dequantize(Tensor codes, Tensor scales, int k) -> Tensor");
  m.def("mx_gemm(Tensor a, Tensor a_scales, Tensor w, Tensor w_scales, Tensor? bias, bool out_f32) -> Tensor");
  m.def("mx_linear(Tensor x, Tensor w, Tensor w_scales, Tensor? bias, int fmt, bool out_f32) -> Tensor");
  m.def("silu_mul_mx(Tensor gate, Tensor up, int fmt) -> (Tensor, Tensor)");
  m.def("rms_norm_modulate_mx(Tensor x, Tensor weight, Tensor shift, float eps, int fmt) -> (Tensor, Tensor)");
  m.def(
      "residual_rms_norm_modulate_mx(Tensor x, Tensor v, Tensor gate, Tensor weight, Tensor shift, float eps, int fmt) "
      "-> (Tensor, Tensor, Tensor)");
  m.def("fp8_quantize(Tensor x) -> (Tensor, Tensor)");
  m.def("fp8_gemm(Tensor a, Tensor a_scales, Tensor w, Tensor w_scales, Tensor? bias) -> Tensor");
  m.def("fp8_linear(Tensor x, Tensor w, Tensor w_scales, Tensor? bias) -> Tensor");
  m.def(
      "qk_norm_rope(Tensor q, Tensor k, Tensor? q_weight, Tensor? k_weight, Tensor cos, Tensor sin, float eps, "
      "Tensor? positions, bool interleaved) -> (Tensor, Tensor)");
  m.def(
      "kv8_append(Tensor k, Tensor v, Tensor cu_seqlens, Tensor lengths, Tensor block_table, Tensor(a!) k_codes, "
      "Tensor(b!) v_codes, Tensor(c!) scales) -> ()");
  m.def(
      "kv8_attention(Tensor q, Tensor cu_seqlens, Tensor lengths, Tensor block_table, Tensor k_codes, Tensor v_codes, "
      "Tensor scales, float scale, bool causal) -> Tensor");
}
TORCH_LIBRARY_IMPL(svdq, CUDA, m) {
  m.impl("linear", TORCH_FN(linear));
  m.impl("linear_siblings", TORCH_FN(linear_siblings));
  m.impl("mx_quantize", TORCH_FN(mx_quantize));
  m.impl("mx_dequantize", TORCH_FN(mx_dequantize));
  m.impl("mx_gemm", TORCH_FN(mx_gemm));
  m.impl("mx_linear", TORCH_FN(mx_linear));
  m.impl("silu_mul_mx", TORCH_FN(silu_mul_mx));
  m.impl("rms_norm_modulate_mx", TORCH_FN(rms_norm_modulate_mx));
  m.impl("residual_rms_norm_modulate_mx", TORCH_FN(residual_rms_norm_modulate_mx));
  m.impl("fp8_quantize", TORCH_FN(fp8_quantize));
  m.impl("fp8_gemm", TORCH_FN(fp8_gemm));
  m.impl("fp8_linear", TORCH_FN(fp8_linear));
  m.impl("qk_norm_rope", TORCH_FN(qk_norm_rope));
  m.impl("kv8_append", TORCH_FN(kv8_append));
  m.impl("kv8_attention", TORCH_FN(kv8_attention));
}
TORCH_LIBRARY_IMPL(svdq, Autograd, m) {
  m.impl("linear", torch::autograd::autogradNotImplementedFallback());
  m.impl("linear_siblings", torch::autograd::autogradNotImplementedFallback());
  m.impl("mx_quantize", torch::autograd::autogradNotImplementedFallback());
  m.impl("mx_dequantize", torch::autograd::autogradNotImplementedFallback());
  m.impl("mx_gemm", torch::autograd::autogradNotImplementedFallback());
  m.impl("mx_linear", torch::autograd::autogradNotImplementedFallback());
  m.impl("silu_mul_mx", torch::autograd::autogradNotImplementedFallback());
  m.impl("rms_norm_modulate_mx", torch::autograd::autogradNotImplementedFallback());
  m.impl("residual_rms_norm_modulate_mx", torch::autograd::autogradNotImplementedFallback());
  m.impl("fp8_quantize", torch::autograd::autogradNotImplementedFallback());
  m.impl("fp8_gemm", torch::autograd::autogradNotImplementedFallback());
  m.impl("fp8_linear", torch::autograd::autogradNotImplementedFallback());
  m.impl("qk_norm_rope", torch::autograd::autogradNotImplementedFallback());
  m.impl("kv8_append", torch::autograd::autogradNotImplementedFallback());
  m.impl("kv8_attention", torch::autograd::autogradNotImplementedFallback());
}
