"""The operators of an attention layer in 8-bit floating point as timed cases:

* ``linear``:  a bf16 activation through a linear layer whose weight is held in E4M3 with a float32 scale for each block
  of 128 x 128 (as 8-bit checkpoints hold it), the activation quantised by the call to E4M3 with a scale for 128
  columns of a row;
* ``product``: the same from an activation that is quantised already;
* ``qk``:      the norms of queries and keys for each head, with a learned weight and the position rotation;
* ``append``:  new keys and values into a cache of E4M3 pages of 64 tokens with a scale for each page and head;
* ``attend``:  attention over such a cache, for a batch of sequences of their own lengths.

The quantisers' scale is the smallest power of two, 2^-126 at least, under which the largest magnitude is at most 448;
codes are the nearest values, ties to even.  Rows are padded with zero codes to a multiple of 128 columns; an activation's
scales are [blocks, rows].  A page's keys are [64, dim], its values [dim, 64]; a page that holds tokens
already keeps its scale unless the new ones need a larger one, and then its older codes are rounded again under that.

Layer sizes are those of the denoiser's linears (hidden 6144, MLP 16384) and of its attention (48 query heads over 12
key / value heads of 128); row counts go from one token to a 1024-pixel image's 4096 latent tokens with 256 text tokens.
"""
from __future__ import annotations

import math
import random

import torch

own = False

HIDDEN, MLP, TOKENS, PAGE = 6144, 16384, 4352, 64
EPS = 1e-6


def _attend(name, batch, q, length, heads, kv, dim, causal, mix):
    return {"name": name, "kind": "attend", "batch": batch, "q": q, "len": length, "heads": heads, "kv": kv, "dim": dim,
            "causal": causal, "mix": mix}


def listed():
    return [
        # one token through a square projection: bound by latency and the weight's bytes
        {"name": "linear token", "kind": "linear", "m": 1, "n": HIDDEN, "k": HIDDEN, "bias": True},
        # a 77-token prompt through a square projection
        {"name": "linear prompt", "kind": "linear", "m": 77, "n": HIDDEN, "k": HIDDEN, "bias": False},
        # odd sizes on every side
        {"name": "product ragged", "kind": "product", "m": 333, "n": 1001, "k": 1187, "bias": True},
        # an image through the MLP's up projection: the largest product
        {"name": "product image", "kind": "product", "m": TOKENS, "n": MLP, "k": HIDDEN, "bias": False},
        # an image's queries and keys, heads sliced from one fused projection
        {"name": "qk image", "kind": "qk", "t": TOKENS, "heads": 48, "kv": 12, "dim": 128, "weights": True, "wide": True,
         "pairs": False, "positions": False},
        # one token for each of 32 sequences, each at a position of its own, neighbouring channels rotated together
        {"name": "qk tokens", "kind": "qk", "t": 32, "heads": 16, "kv": 4, "dim": 64, "weights": True, "wide": False,
         "pairs": True, "positions": True},
        # three prompts into the cache, behind what it holds of them
        {"name": "append prompts", "kind": "append", "batch": 3, "q": 1101, "len": 2381, "kv": 12, "dim": 128, "mix": 3},
        # one token for each of 32 sequences
        {"name": "append tokens", "kind": "append", "batch": 32, "q": 1, "len": 8192, "kv": 12, "dim": 128, "mix": 1},
        # one token over a long cache: the cache's bytes, split over the card
        _attend("attend token", 1, 1, 131072, 48, 12, 128, True, 0),
        # a batch of sequences of any length up to 8192, one token each
        _attend("attend tokens", 32, 1, 8192, 48, 12, 128, True, 2),
        # the next chunk of three prompts, causal, heads of 64
        _attend("attend chunk", 3, 777, 5000, 16, 4, 64, True, 4),
        # an image's latent and text tokens over themselves and 256 tokens that the cache held: all of it visible
        _attend("attend image", 1, TOKENS, TOKENS + 256, 48, 12, 128, False, 0),
    ]


def draw(rng):
    def size(lo, hi):
        return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))

    kind = rng.choice(["linear", "product", "qk", "append", "attend", "attend"])
    if kind in ("linear", "product"):
        step = rng.choice([1, 8, 128])
        case = {"kind": kind, "m": size(1, TOKENS), "n": size(64, MLP), "k": -(-size(64, MLP) // step) * step,
                "bias": rng.random() < 0.5}
        while case["m"] * case["n"] * case["k"] > TOKENS * MLP * HIDDEN:
            case["n"] = max(64, case["n"] // 2)
        return case
    kv = rng.choice([1, 2, 4, 8, 12])
    if kind == "qk":
        return {"kind": kind, "t": size(1, TOKENS), "heads": kv * rng.choice([1, 2, 3, 4]), "kv": kv,
                "dim": rng.choice([64, 96, 128, 256]), "weights": rng.random() < 0.7, "wide": rng.random() < 0.5,
                "pairs": rng.random() < 0.5, "positions": rng.random() < 0.5}
    case = {"kind": kind, "batch": size(1, 32), "q": 1 if rng.random() < 0.4 else size(1, TOKENS), "len": size(1, 32768),
            "kv": kv, "dim": rng.choice([64, 128]), "mix": rng.randrange(1, 10 ** 6)}
    case["len"] = max(case["len"], case["q"])
    if kind == "attend":
        case |= {"heads": kv * rng.choice([1, 2, 3, 4, 7, 8]), "causal": rng.random() < 0.7}
    while (case["batch"] * (case["len"] + PAGE) * kv * case["dim"] > 4e8 or
           case["batch"] * case["q"] * case["len"] * case.get("heads", 0) > 9e8):
        if case["batch"] > 1:
            case["batch"] = (case["batch"] + 1) // 2
        else:
            case["len"], case["q"] = (case["len"] + 1) // 2, (case["q"] + 1) // 2
    return case


def _ragged(case):
    """(new tokens, tokens held when they are in) of each sequence: the largest of each for the first, for the others
    anything up to them, now and then nothing new.  mix 0: all of them the largest."""
    rng, out = random.Random(case["mix"]), []
    for b in range(case["batch"]):
        n, length = case["q"], case["len"]
        if b and case["mix"]:
            n = 0 if rng.random() < 0.1 else rng.randint(1, n)
            length = rng.randint(n, length)
        out.append((n, length))
    return out


# ---- what a program holds before the calls ----
def _activation(shape, gen):
    """A bf16 activation: unit normal values with a few channels that are 8 to 24 times larger."""
    x = torch.randn(shape, device="cuda", generator=gen)
    big = torch.rand(shape[-1], device="cuda", generator=gen) < 0.01
    amp = torch.where(big, 8 + 16 * torch.rand(shape[-1], device="cuda", generator=gen), torch.ones((), device="cuda"))
    return (x * amp).to(torch.bfloat16)


def _pow2(amax):
    """The smallest power of two s >= 2^-126 with amax <= 448 s."""
    m, e = torch.frexp(amax)                      # amax = m 2^e, m in [0.5, 1); 448 = 0.875 2^9
    e = torch.where(m <= 0.875, e - 9, e - 8)
    return torch.ldexp(torch.ones((), device=amax.device, dtype=amax.dtype), torch.where(amax > 0, e, -126).clamp_min(-126))


def _encode_rows(x):
    """f32 [M, K] -> E4M3 codes [M, K padded to 128] and f32 scales [blocks, M]."""
    x = torch.nn.functional.pad(x, (0, -x.shape[1] % 128))
    b = x.view(x.shape[0], -1, 128)
    s = _pow2(b.abs().amax(-1))
    return (b / s[..., None]).to(torch.float8_e4m3fn).view(x.shape), s.T.contiguous()


def _weight(n, k, gen):
    """An E4M3 weight [n, k padded to 128] with float32 scales for blocks of 128 x 128, of N(0, 0.02) values."""
    w = torch.randn((n, k), device="cuda", generator=gen) * 0.02
    w = torch.nn.functional.pad(w, (0, -k % 128, 0, -n % 128))
    b = w.view(w.shape[0] // 128, 128, -1, 128)
    s = b.abs().amax((1, 3)) / 448
    codes = (b / s[:, None, :, None]).to(torch.float8_e4m3fn).view(w.shape)
    return codes[:n].contiguous(), s


def _pages(shape, gen):
    """A cache of pages in E4M3: keys [pages, kv, 64, dim] with a few larger channels, values [pages, kv, dim, 64], and
    their scales [pages, kv, 2]."""
    pages, kv, dim = shape
    k = _activation((pages, kv, PAGE, dim), gen).float()
    v = _activation((pages, kv, dim, PAGE), gen).float()
    s = torch.stack([_pow2(x.abs().amax((2, 3))) for x in (k, v)], -1)
    return ((k / s[..., :1, None]).to(torch.float8_e4m3fn), (v / s[..., 1:, None]).to(torch.float8_e4m3fn), s)


def _cache(s, case, gen):
    """The cache's pages in any order, its table (-1 behind a sequence's last page), lengths and new tokens' offsets."""
    seqs = _ragged(case)
    need = [-(-length // PAGE) for _, length in seqs]
    order = torch.randperm(sum(need) + 4, device="cuda", generator=gen).to(torch.int32)
    table = torch.full((len(seqs), max(need) + 1), -1, dtype=torch.int32, device="cuda")
    first = 0
    for b, n in enumerate(need):
        table[b, :n] = order[first:first + n]
        first += n
    s["table"] = table
    s["k_codes"], s["v_codes"], s["scales"] = _pages((len(order), case["kv"], case["dim"]), gen)
    offsets = [sum(n for n, _ in seqs[:b]) for b in range(len(seqs) + 1)]
    s["offsets"] = torch.tensor(offsets, dtype=torch.int32, device="cuda")
    s["rows"], s["most"] = offsets[-1], max(n for n, _ in seqs)
    held = [length - (n if case["kind"] == "append" else 0) for n, length in seqs]
    s["lengths"] = torch.tensor(held, dtype=torch.int32, device="cuda")


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    kind, s = case["kind"], dict(case)
    if kind in ("linear", "product"):
        x = _activation((case["m"], case["k"]), gen)
        s["w"], s["ws"] = _weight(case["n"], case["k"], gen)
        s["b"] = torch.randn(case["n"], device="cuda", generator=gen).to(torch.bfloat16) if case["bias"] else None
        if kind == "linear":
            s["x"] = x
        else:
            s["a"], s["as"] = _encode_rows(x.float())
    elif kind == "qk":
        t, dim, heads, kv = case["t"], case["dim"], case["heads"], case["kv"]
        x = _activation((t, heads + 2 * kv, dim), gen)      # a fused projection: queries, keys, values
        s["q"], s["k"] = x[:, :heads], x[:, heads:heads + kv]
        s["qw"], s["kw"] = ((1 + 0.2 * torch.randn((2, dim), device="cuda", generator=gen)).to(torch.bfloat16).unbind(0)
                            if case["weights"] else (None, None))
        far = 32768 if case["positions"] else t
        inv = 10000.0 ** (-torch.arange(0, dim, 2, device="cuda", dtype=torch.float64) / dim)
        angle = torch.arange(far, device="cuda", dtype=torch.float64)[:, None] * inv
        s["cos"], s["sin"] = (f(angle).to(torch.float32 if case["wide"] else torch.bfloat16) for f in (torch.cos, torch.sin))
        s["at"] = torch.randint(0, far, (t,), device="cuda", generator=gen) if case["positions"] else None
    else:
        _cache(s, case, gen)
        if kind == "append":
            s["k"], s["v"] = (_activation((s["rows"], case["kv"], case["dim"]), gen) for _ in range(2))
        else:
            s["q"] = _activation((s["rows"], case["heads"], case["dim"]), gen)
    return s


# ---- the plain forms ----
def _product(a, a_scales, s):
    """The products and sums of a layer in float32, rounded once."""
    kb = a.shape[1] // 128
    a = (a.float().view(a.shape[0], kb, 128) * a_scales.T[..., None]).view(a.shape)
    ws = s["ws"].repeat_interleave(128, 0)[:s["n"]]
    w = (s["w"].float().view(s["n"], kb, 128) * ws[..., None]).view(s["w"].shape)
    y = a @ w.T
    return (y if s["b"] is None else y + s["b"].float()).to(torch.bfloat16)


def _norm_rope(x, weight, s):
    x = x.float()
    x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS)
    if weight is not None:
        x = x * weight.float()
    c, n = (t[:x.shape[0]] if s["at"] is None else t[s["at"]] for t in (s["cos"], s["sin"]))
    c, n = c.float()[:, None], n.float()[:, None]
    if s["pairs"]:
        a, b = x[..., 0::2], x[..., 1::2]
        return torch.stack([a * c - b * n, b * c + a * n], -1).flatten(-2).to(torch.bfloat16)
    a, b = x.chunk(2, -1)
    return torch.cat([a * c - b * n, b * c + a * n], -1).to(torch.bfloat16)


def _rows(s):
    """Of each new token: its sequence, and how many of that sequence's new tokens precede it."""
    at = torch.arange(s["rows"], device="cuda")
    seq = torch.searchsorted(s["offsets"][1:].long(), at, right=True)
    return seq, at - s["offsets"].long()[seq]


def _store(s):
    """The new tokens into their pages, in place."""
    seq, i = _rows(s)
    held = s["lengths"].long()[seq]
    place = held + i
    page, slot = s["table"].long()[seq, place // PAGE], place % PAGE
    older = held - place // PAGE * PAGE                     # tokens that the page held before: > 0 in a page begun earlier
    touched, where = page.unique(return_inverse=True)
    keep = torch.zeros(len(touched), dtype=torch.long, device="cuda").index_copy_(0, where, older.clamp(0, PAGE))
    slots = torch.arange(PAGE, device="cuda") < keep[:, None]
    scales = s["scales"]
    for c, (x, codes) in enumerate(((s["k"].float(), s["k_codes"]), (s["v"].float(), s["v_codes"]))):
        amax = torch.zeros((len(touched), x.shape[1]), device="cuda")
        amax.index_reduce_(0, where, x.abs().amax(-1), "amax")
        before = scales[touched, :, c]
        after = torch.where(keep[:, None] > 0, torch.maximum(before, _pow2(amax)), _pow2(amax))
        old = codes[touched]
        again = (old.float() * (before / after)[..., None, None]).to(torch.float8_e4m3fn)
        mask = slots[:, None, :, None] if c == 0 else slots[:, None, None, :]
        new = torch.where(mask, again.view(torch.uint8), old.view(torch.uint8))
        bits = (x / after[where][..., None]).to(torch.float8_e4m3fn).view(torch.uint8)
        if c == 0:
            new[where, :, slot] = bits
        else:
            new[where, :, :, slot] = bits
        codes.view(torch.uint8)[touched] = new
        scales[touched, :, c] = after
    return s["k_codes"], s["v_codes"], scales


def _attention(s):
    seq, i = _rows(s)
    batch, heads, kv, dim, most = s["batch"], s["heads"], s["kv"], s["dim"], s["most"]
    q = torch.zeros((batch, most, kv, heads // kv, dim), device="cuda")
    q[seq, i] = s["q"].float().view(-1, kv, heads // kv, dim)
    q = q.permute(0, 2, 1, 3, 4).reshape(batch, kv, -1, dim)
    pages = s["table"].long().clamp_min(0)
    scales = s["scales"][pages]                             # [batch, pages, kv, 2]
    k = (s["k_codes"][pages].float() * scales[..., :1, None]).transpose(1, 2).reshape(batch, kv, -1, dim)
    v = (s["v_codes"][pages].float() * scales[..., 1:, None]).permute(0, 2, 1, 4, 3).reshape(batch, kv, -1, dim)
    length = s["lengths"].long()[:, None, None]
    new = (s["offsets"][1:] - s["offsets"][:-1]).long()[:, None, None]
    key = torch.arange(k.shape[2], device="cuda")
    last = length - new + torch.arange(most, device="cuda")[None, :, None] if s["causal"] else length - 1
    seen = ((key <= last) & (key < length)).expand(batch, most, -1)
    seen = seen.repeat_interleave(heads // kv, 1)[:, None]
    p = (q @ k.transpose(2, 3)).mul_(dim ** -0.5).masked_fill_(~seen, -math.inf)
    top = p.amax(-1, keepdim=True)
    p = p.sub_(torch.where(top == -math.inf, 0.0, top)).exp_()
    total = p.sum(-1, keepdim=True)
    o = (p @ v) / torch.where(total == 0, 1.0, total)
    o = o.view(batch, kv, most, -1, dim).permute(0, 2, 1, 3, 4).reshape(batch, most, heads, dim)
    return o[seq, i].to(torch.bfloat16)


def run(state):
    """One call of the operator."""
    s, kind = state, state["kind"]
    if own:
        from krea2_svdquant_amd.kernels.hip import ops
        if kind == "linear":
            return ops.fp8_linear(s["x"], s["w"], s["ws"], s["b"])
        if kind == "product":
            return ops.fp8_gemm(s["a"], s["as"], s["w"], s["ws"], s["b"])
        if kind == "qk":
            return ops.qk_norm_rope(s["q"], s["k"], s["qw"], s["kw"], s["cos"], s["sin"], EPS, s["at"], s["pairs"])
        cache = (s["offsets"], s["lengths"], s["table"], s["k_codes"], s["v_codes"], s["scales"])
        if kind == "append":
            ops.kv8_append(s["k"], s["v"], *cache)
            return cache[3:]
        return ops.kv8_attention(s["q"], *cache, s["dim"] ** -0.5, s["causal"])
    if kind == "linear":
        return _product(*_encode_rows(s["x"].float()), s)
    if kind == "product":
        return _product(s["a"], s["as"], s)
    if kind == "qk":
        return _norm_rope(s["q"], s["qw"], s), _norm_rope(s["k"], s["kw"], s)
    if kind == "append":
        return _store(s)
    return _attention(s)


def work(case):
    kind = case["kind"]
    if kind in ("linear", "product"):
        m, n, k = case["m"], case["n"], case["k"]
        held = 2 if kind == "linear" else 1 + 4 / 128
        return {"bytes": m * k * held + n * k * (1 + 4 / 128 ** 2) + 2 * m * n + (2 * n if case["bias"] else 0),
                "flops": 2.0 * m * n * k}
    if kind == "qk":
        values = case["t"] * (case["heads"] + case["kv"]) * case["dim"]
        return {"bytes": 4 * values + case["t"] * case["dim"] * (4 if case["wide"] else 2), "flops": 8.0 * values}
    seqs = _ragged(case)
    rows, width = sum(n for n, _ in seqs), case["kv"] * case["dim"]
    if kind == "append":    # keys and values in bf16 in, in 8 bits out
        return {"bytes": rows * width * 2 * (2 + 1), "flops": 4.0 * rows * width}
    wide = case["heads"] * case["dim"]
    pairs = sum(n * length - (n * (n - 1) // 2 if case["causal"] else 0) for n, length in seqs)
    read = sum(length for n, length in seqs if n)
    return {"bytes": 2 * read * width + 4 * rows * wide, "flops": 4.0 * pairs * wide}


# ---- the definition in 64 bits ----
def _round64(x):
    """float64 values at the nearest E4M3 value, ties to even."""
    mag = x.abs()
    step = torch.exp2(torch.floor(torch.log2(mag.clamp_min(2.0 ** -6))) - 3)
    return torch.sign(x) * (torch.round(mag / step) * step).clamp_max(448.0)


def _scale64(top):
    """The smallest power of two from 2^-126 with top <= 448 of it."""
    e = torch.ceil(torch.log2(top.clamp_min(2.0 ** -140) / 448)).clamp_min(-126.0)
    return torch.exp2(torch.where(top > 448 * torch.exp2(e), e + 1, e))


def exact(case, seed):
    s, kind = prepare(case, seed), case["kind"]
    if kind in ("linear", "product"):
        kb = s["w"].shape[1] // 128
        if kind == "linear":
            x = s["x"].double()
            x = torch.cat([x, x.new_zeros(len(x), kb * 128 - x.shape[1])], 1).reshape(len(x), kb, 128)
            scale = _scale64(x.abs().max(-1).values)[..., None]
            a = (_round64(x / scale) * scale).reshape(len(x), -1)
        else:
            a = (s["a"].double().reshape(-1, kb, 128) * s["as"].double().T[..., None]).reshape(s["a"].shape)
        block = torch.arange(case["n"], device="cuda") // 128
        w = (s["w"].double().reshape(-1, kb, 128) * s["ws"].double()[block][..., None]).reshape(s["w"].shape)
        y = torch.cat([part @ w.T for part in a.split(1024)])
        return y if s["b"] is None else y + s["b"].double()
    if kind == "qk":
        at = torch.arange(case["t"], device="cuda") if s["at"] is None else s["at"]
        c, n = s["cos"].double()[at][:, None], s["sin"].double()[at][:, None]
        out = []
        for x, weight in ((s["q"], s["qw"]), (s["k"], s["kw"])):
            x = x.double()
            x = x / torch.sqrt((x * x).sum(-1, keepdim=True) / case["dim"] + EPS) * (1.0 if weight is None else weight.double())
            half = case["dim"] // 2
            first, second = (x[..., ::2], x[..., 1::2]) if case["pairs"] else (x[..., :half], x[..., half:])
            y = torch.empty_like(x)
            a, b = (y[..., ::2], y[..., 1::2]) if case["pairs"] else (y[..., :half], y[..., half:])
            a.copy_(first * c - second * n)
            b.copy_(second * c + first * n)
            out.append(y)
        return tuple(out)
    seqs, table, first = _ragged(case), s["table"].tolist(), 0
    kc, vc, scales = s["k_codes"].double(), s["v_codes"].double(), s["scales"].double()
    if kind == "append":
        for b, (n, length) in enumerate(seqs):
            place = length - n
            while place < length:
                page, slot = table[b][place // PAGE], place % PAGE
                count = min(PAGE - slot, length - place)
                for c, (codes, x) in enumerate(((kc, s["k"]), (vc.transpose(2, 3), s["v"]))):
                    x = x[first:first + count].double().transpose(0, 1)
                    need = _scale64(x.abs().amax((1, 2)))
                    if slot:
                        before = scales[page, :, c].clone()
                        need = torch.maximum(need, before)
                        codes[page, :, :slot] = _round64(codes[page, :, :slot] * (before / need)[:, None, None])
                    codes[page, :, slot:slot + count] = _round64(x / need[:, None, None])
                    scales[page, :, c] = need
                first, place = first + count, place + count
        return kc, vc, scales
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    group = case["heads"] // case["kv"]
    for b, (n, length) in enumerate(seqs):
        pages = torch.tensor(table[b][:-(-length // PAGE)], device="cuda", dtype=torch.long)
        for h in range(case["kv"] if n and length else 0):
            k = (kc[pages, h] * scales[pages, h, 0][:, None, None]).reshape(-1, case["dim"])[:length]
            v = (vc[pages, h] * scales[pages, h, 1][:, None, None]).transpose(1, 2).reshape(-1, case["dim"])[:length]
            for g in range(h * group, (h + 1) * group):
                p = s["q"][first:first + n, g].double() @ k.T / math.sqrt(case["dim"])
                if case["causal"]:
                    p += torch.full_like(p, -math.inf).triu(length - n + 1)
                out[first:first + n, g] = torch.softmax(p, -1) @ v
        first += n
    return out
