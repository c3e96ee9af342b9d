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
}
