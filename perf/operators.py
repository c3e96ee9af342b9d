"""The microscaled (MX) operators as timed cases: blocks of 32 values along a row that share a power-of-two
scale (E8M0), held in 4 bits (E2M1, two per byte, the even column in the low half) or 8 bits (E4M3).

* ``quantize``: a bf16 activation into MX blocks, and read back;
* ``product``:  ``a @ w^T + bias`` of an MX activation (4 or 8 bits) with an MX weight (4 bits);
* ``linear``:   the two together, from a bf16 activation to the layer's output;
* ``norm``:     the gated residual add and the adaptive RMS norm, with the normed row in 8 bits with scales;
* ``silu``:     the SwiGLU product, in 8 bits with scales.

The scale of a block is 2^(floor(log2(largest magnitude)) - E), E the exponent of the element type's largest
value (2 for E2M1, 8 for E4M3), its exponent kept within -127..127; elements are rounded to the nearest value
of their type, ties to the even code, beyond its largest value to that.  Rows are padded with zeros to a
multiple of 128 columns, a row's scales to a multiple of 16; a block of zeros has the smallest scale.  Layer sizes are those of the denoiser's
linears (hidden 6144, key / value width 1536, MLP 16384), row counts from one token to a 1024-pixel
image's 4096 latent tokens with 256 text tokens.
"""
from __future__ import annotations

import math

import torch

own = False

HIDDEN, KV, MLP, TOKENS = 6144, 1536, 16384, 4352
EPS = 1e-6
E2M1, E4M3 = "e2m1", "e4m3"
EMAX = {E2M1: 2, E4M3: 8}


def _product(name, m, n, k, fmt, bias=False, f32=False):
    return {"name": name, "kind": "product", "m": m, "n": n, "k": k, "fmt": fmt, "bias": bias, "f32": f32}


def listed():
    return [
        # an image's activation on its way into a 4-bit product
        {"name": "quantize image e2m1", "kind": "quantize", "m": TOKENS, "k": HIDDEN, "fmt": E2M1},
        # a short prompt of a width that no block divides, in 8 bits
        {"name": "quantize prompt e4m3", "kind": "quantize", "m": 77, "k": 1000, "fmt": E4M3},
        # one token through a square projection: the smallest product, bound by latency and the weight's bytes
        _product("product token", 1, HIDDEN, HIDDEN, E4M3, bias=True),
        # a 256-token prompt through the MLP's up projection
        _product("product prompt ff.up", 256, MLP, HIDDEN, E2M1),
        # a handful of rows and odd sizes on every side, 32-bit output
        _product("product ragged", 333, 1001, 1187, E4M3, bias=True, f32=True),
        # an image through the MLP's up projection: the widest product
        _product("product image ff.up", TOKENS, MLP, HIDDEN, E2M1),
        # an image through the MLP's down projection with 8-bit activations: the longest reduction
        _product("product image ff.down", TOKENS, HIDDEN, MLP, E4M3),
        # a 768-pixel image with a 77-token prompt through the key projection, from bf16 to bf16
        {"name": "linear image to_k", "kind": "linear", "m": 2381, "n": KV, "k": HIDDEN, "fmt": E2M1, "bias": False},
        # a 77-token prompt through a square projection with 8-bit activations
        {"name": "linear prompt to_q", "kind": "linear", "m": 77, "n": HIDDEN, "k": HIDDEN, "fmt": E4M3, "bias": True},
        # the norm ahead of a block's MLP over an image with its prompt
        {"name": "norm image", "kind": "norm", "m": TOKENS, "k": HIDDEN},
        # the same for one row
        {"name": "norm token", "kind": "norm", "m": 1, "k": HIDDEN},
        # the SwiGLU product over an image with its prompt
        {"name": "silu image", "kind": "silu", "m": TOKENS, "k": MLP},
    ]


def draw(rng):
    def size(lo, hi, step=1):
        return max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi))) / step)) * step)

    kind = rng.choice(["quantize", "product", "product", "linear", "norm", "silu"])
    step = rng.choice([1, 8, 64])
    case = {"kind": kind, "m": size(1, TOKENS), "k": size(128, MLP, step)}
    if kind == "silu":
        return case
    if kind == "norm":   # rows of whole 16-byte chunks, as the framework's norms take them
        case["k"] = min(HIDDEN * 2, case["k"] + 7) // 8 * 8
        return case
    case["fmt"] = rng.choice([E2M1, E4M3])
    if kind == "quantize":
        return case
    case["n"] = size(64, MLP, rng.choice([1, 8, 64]))
    case["bias"] = rng.random() < 0.5
    while case["m"] * case["n"] * case["k"] > TOKENS * MLP * HIDDEN:
        case["n"] = max(64, case["n"] // 2)
    if kind == "product":
        case["f32"] = rng.random() < 0.25
    return case


def _activation(shape, gen):
    """A bf16 activation: unit normal values with a few channels that are 8 to 24 times larger."""
    x = torch.randn(shape, device="cuda", generator=gen)
    big = torch.rand(shape[-1], device="cuda", generator=gen) < 0.01
    amp = torch.where(big, 8 + 16 * torch.rand(shape[-1], device="cuda", generator=gen), torch.ones((), device="cuda"))
    return (x * amp).to(torch.bfloat16)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    m, k, kind = case["m"], case["k"], case["kind"]
    s = dict(case)
    if kind == "norm":
        s["x"], s["v"] = _activation((m, k), gen), _activation((m, k), gen)
        s["gate"], s["weight"], s["shift"] = (
            (a + b * torch.randn(k, device="cuda", generator=gen)).to(torch.bfloat16) for a, b in ((0.5, 0.2), (1, 0.1), (0, 0.1)))
        return s
    if kind == "silu":
        s["gate"], s["up"] = _activation((m, k), gen), _activation((m, k), gen)
        return s
    x = _activation((m, k), gen)
    if kind == "quantize":
        s["x"] = x
        return s
    n = case["n"]
    w = torch.randn((n, k), device="cuda", generator=gen) * 0.02
    s["w"], s["ws"] = _encode(w, E2M1)
    s["bias"] = torch.randn(n, device="cuda", generator=gen).to(torch.bfloat16) if case["bias"] else None
    if kind == "linear":
        s["x"] = x
    else:
        s["a"], s["as"] = _encode(x.float(), case["fmt"])
    return s


# ---- the plain forms ----
def _pad(x):
    k = x.shape[1]
    return torch.nn.functional.pad(x, (0, -k % 128))


def _encode(x, fmt):
    """f32 [M, K] -> codes (uint8 [M, Kp / 2] or float8_e4m3fn [M, Kp]) and scales (float8_e8m0fnu, a
    row's padded to whole 16 bytes)."""
    x = _pad(x)
    b = x.view(x.shape[0], -1, 32)
    amax = b.abs().amax(-1)
    e = torch.frexp(amax).exponent - 1 - EMAX[fmt]
    e = torch.where(amax > 0, e, -127).clamp(-127, 127)
    v = torch.ldexp(b, -e[..., None]).view(x.shape)
    scales = torch.nn.functional.pad((e + 127).to(torch.uint8), (0, -e.shape[1] % 16)).view(torch.float8_e8m0fnu)
    if fmt == E4M3:
        return v.clamp(-448, 448).to(torch.float8_e4m3fn), scales
    a = v.abs()
    code = ((a > 0.25).byte() + (a >= 0.75).byte() + (a > 1.25).byte() + (a >= 1.75).byte() + (a > 2.5).byte()
            + (a >= 3.5).byte() + (a > 5).byte() + torch.signbit(v).byte() * 8)
    return code[:, 0::2] | (code[:, 1::2] << 4), scales


def _decode(codes, scales):
    """f32 values of MX codes, padding included."""
    if codes.dtype == torch.uint8:
        c = torch.stack([codes & 15, codes >> 4], -1).flatten(1)
        table = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], device=codes.device)
        v = torch.where(c >= 8, -1.0, 1.0) * table[(c & 7).int()]
    else:
        v = codes.float()
    s = scales.view(torch.uint8)[:, :v.shape[1] // 32].int() - 127
    s = torch.ldexp(torch.ones((), device=codes.device), s)
    return (v.view(v.shape[0], -1, 32) * s[..., None]).view(v.shape)


def _matmul(a, a_scales, w, w_scales, bias, f32):
    y = _decode(a, a_scales) @ _decode(w, w_scales).T
    if bias is not None:
        y = y + bias.float()
    return y if f32 else y.to(torch.bfloat16)


def _plain(s):
    kind = s["kind"]
    if kind == "quantize":
        return _decode(*_encode(s["x"].float(), s["fmt"]))[:, :s["k"]].to(torch.bfloat16)
    if kind == "product":
        return _matmul(s["a"], s["as"], s["w"], s["ws"], s["bias"], s["f32"])
    if kind == "linear":
        return _matmul(*_encode(s["x"].float(), s["fmt"]), s["w"], s["ws"], s["bias"], False)
    if kind == "norm":
        x = (s["x"].float() + s["gate"].float() * s["v"].float()).to(torch.bfloat16)
        f = x.float()
        y = f * torch.rsqrt(f.square().mean(-1, keepdim=True) + EPS) * s["weight"].float() + s["shift"].float()
        return (x, *_encode(y, E4M3))
    g = s["gate"].float()
    return _encode(g / (1 + torch.exp(-g)) * s["up"].float(), E4M3)


def run(state):
    """One call of the operator.  Quantized values come back as bf16 (read back; exact in bf16) or as the
    float8 tensors that hold them."""
    s = state
    if not own:
        return _plain(s)
    from krea2_svdquant_amd.kernels.hip import ops
    kind = s["kind"]
    if kind == "quantize":
        return ops.mx_dequantize(*ops.mx_quantize(s["x"], s["fmt"]), s["k"])
    if kind == "product":
        return ops.mx_gemm(s["a"], s["as"], s["w"], s["ws"], s["bias"], s["f32"])
    if kind == "linear":
        return ops.mx_linear(s["x"], s["w"], s["ws"], s["bias"], s["fmt"])
    if kind == "norm":
        return ops.residual_rms_norm_modulate_mx(s["x"], s["v"], s["gate"], s["weight"], s["shift"], EPS, E4M3)
    return ops.silu_mul_mx(s["gate"], s["up"], E4M3)


def work(case):
    m, k, kind = case["m"], case["k"], case["kind"]
    held = {E2M1: 0.5 + 1 / 32, E4M3: 1 + 1 / 32}   # bytes per value, its share of the scale included
    if kind == "quantize":    # read, write the codes, read them back, write the values
        return {"bytes": m * k * (2 + 2 * held[case["fmt"]] + 2), "flops": 4.0 * m * k}
    if kind == "norm":        # x, v in; the new residual and the codes out; three vectors
        return {"bytes": m * k * (2 + 2 + 2 + held[E4M3]) + 6 * k, "flops": 9.0 * m * k}
    if kind == "silu":
        return {"bytes": m * k * (2 + 2 + held[E4M3]), "flops": 8.0 * m * k}
    n = case["n"]
    a = 2 if kind == "linear" else held[case["fmt"]]
    out = 4 if case.get("f32") else 2
    return {"bytes": m * k * a + n * k * held[E2M1] + m * n * out + (2 * n if case["bias"] else 0),
            "flops": 2.0 * m * n * k}


# ---- the definition in 64 bits ----
def _held64(x, fmt):
    """What float64 values become in MX blocks: (values without the scale, scales), padded."""
    x = torch.cat([x, x.new_zeros(x.shape[0], -x.shape[1] % 128)], 1)
    blocks = x.reshape(x.shape[0], -1, 32)
    top = blocks.abs().max(-1).values
    scale = torch.exp2((torch.floor(torch.log2(top)) - EMAX[fmt]).clamp(-127, 127))   # log2(0): the smallest
    v = blocks / scale[..., None]
    bits, low, most = (1, 0, 6.0) if fmt == E2M1 else (3, -6, 448.0)
    mag = v.abs()
    # the spacing of the element type's values around each magnitude
    step = torch.exp2(torch.floor(torch.log2(mag.clamp_min(2.0 ** low))) - bits)
    q = torch.round(mag / step) * step
    scale = torch.cat([scale, scale.new_full((len(scale), -scale.shape[1] % 16), 2.0 ** -127)], 1)
    return (torch.sign(v) * q.clamp_max(most)).reshape(x.shape), scale


def _times64(q, scale):
    return (q.reshape(q.shape[0], -1, 32) * scale[:, :q.shape[1] // 32, None]).reshape(q.shape)


def exact(case, seed):
    s = prepare(case, seed)
    kind, k = case["kind"], case["k"]
    if kind == "quantize":
        return _times64(*_held64(s["x"].double(), case["fmt"]))[:, :k]
    if kind == "norm":
        x = (s["x"].double() + s["gate"].double() * s["v"].double()).to(torch.bfloat16).double()
        r = 1 / torch.sqrt((x * x).sum(-1, keepdim=True) / k + EPS)
        return (x, *_held64(x * r * s["weight"].double() + s["shift"].double(), E4M3))
    if kind == "silu":
        g = s["gate"].double()
        return _held64(g * torch.sigmoid(g) * s["up"].double(), E4M3)
    grid = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6, -0.0, -0.5, -1, -1.5, -2, -3, -4, -6], device="cuda",
                        dtype=torch.float64)

    def values(codes, scales):
        if codes.dtype == torch.uint8:
            v = codes.new_empty((codes.shape[0], codes.shape[1] * 2), dtype=torch.float64)
            v[:, 0::2], v[:, 1::2] = grid[(codes % 16).long()], grid[(codes // 16).long()]
        else:
            v = codes.double()
        return _times64(v, scales.double())

    a = _times64(*_held64(s["x"].double(), case["fmt"])) if kind == "linear" else values(s["a"], s["as"])
    w = values(s["w"], s["ws"])
    y = torch.cat([p @ w.T for p in a.split(1024)])
    return y if s["bias"] is None else y + s["bias"].double()
