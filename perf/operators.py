"""The block-scaled 8-bit floating-point linear and the query / key preparation: what is measured.

Four operators, in the order a transformer block uses them:

* ``quantize``  activations to e4m3 with one power-of-two (e8m0) scale for each row's group of 128;
* ``weight``    a weight to e4m3 with one such scale for each block of 128 x 128;
* ``matmul``    the product of the two, with the linear's output stage (bias, activation, gate, residual);
* ``qk``        RMS norm of each query and key head, rotation by position, heads moved in front of tokens.

With ``own`` false the functions below compute them from elementary torch operations; with ``own``
true they call the ``sdq`` package.  Sizes are those of the layers in ``sdq/encoders.py`` and
``sdq/flux.py``, and ragged ones.
"""
from __future__ import annotations

import math
import os
import sys

import torch

own = False

BLOCK = 128          # values that share a scale: along a row (activations), both ways (weights)
MAX_E4M3 = 448.0
_DT = {"bf16": torch.bfloat16, "f32": torch.float32}


def _sdq():
    path = os.path.join(os.getcwd(), "stable-diffusion.rs_b200")
    if path not in sys.path:
        sys.path.insert(0, path)
    import sdq

    return sdq


# ---------------------------------------------------------------- cases
def listed():
    return [
        # One prompt of 512 tokens entering a T5-XXL layer: launch-bound.
        {"name": "quantize prompt", "op": "quantize", "m": 512, "k": 4096, "dtype": "bf16"},
        # Flux's joint sequence (512 text + 4096 image tokens) before an MLP's down projection.
        {"name": "quantize image mlp", "op": "quantize", "m": 4608, "k": 12288, "dtype": "bf16"},
        # f32 activations, odd row count, a row that ends inside a group.
        {"name": "quantize ragged f32", "op": "quantize", "m": 1037, "k": 2640, "dtype": "f32"},
        # Load time: a grouped-query key projection (Qwen3-4B), and the largest MLP matrix (Mistral Small).
        {"name": "weight small", "op": "weight", "n": 1024, "k": 2560, "dtype": "bf16"},
        {"name": "weight large", "op": "weight", "n": 32768, "k": 5120, "dtype": "bf16"},
        # One token through an MLP's up projection (Qwen3-4B): the weight's bytes and latency.
        {"name": "matmul one token", "op": "matmul", "m": 1, "k": 2560, "n": 9728, "act": "", "extra": False},
        # A few conditioning rows at once, SiLU in the output stage (Qwen2.5-VL widths).
        {"name": "matmul five rows silu", "op": "matmul", "m": 5, "k": 3584, "n": 18944, "act": "silu", "extra": False},
        # Odd everything, with gate and residual: ragged tiles on each side, an unaligned output pitch.
        {"name": "matmul ragged gated", "op": "matmul", "m": 333, "k": 2640, "n": 4099, "act": "", "extra": True},
        # A prompt through T5-XXL's first MLP layer, GELU.
        {"name": "matmul prompt gelu", "op": "matmul", "m": 512, "k": 4096, "n": 10240, "act": "gelu_approx",
         "extra": False},
        # Image-sized rows through the largest MLP matrix: the tensor cores' rate.
        {"name": "matmul large", "op": "matmul", "m": 4096, "k": 5120, "n": 32768, "act": "", "extra": False},
        # Flux's joint attention: 24 heads, interleaved pairs, cut out of a wider projection.
        {"name": "qk image", "op": "qk", "b": 1, "n": 4608, "heads": 24, "kv": 24, "d": 128, "rope": 128, "pad": 12288,
         "pairs": "interleaved", "dtype": "bf16", "positions": False},
        # Eight sequences decoding one token each at their own positions, grouped heads, half-split pairs.
        {"name": "qk one token", "op": "qk", "b": 8, "n": 1, "heads": 32, "kv": 8, "d": 128, "rope": 128, "pad": 0,
         "pairs": "halves", "dtype": "bf16", "positions": True},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["quantize", "weight", "matmul", "matmul", "matmul", "qk", "qk"])
    if op == "quantize":
        return {"op": op, "m": _log(rng, 1, 4608), "k": 16 * _log(rng, 1, 768), "dtype": rng.choice(["bf16", "bf16", "f32"])}
    if op == "weight":
        return {"op": op, "n": _log(rng, 1, 16384), "k": 16 * _log(rng, 1, 512), "dtype": rng.choice(["bf16", "f32"])}
    if op == "matmul":
        return {"op": op, "m": _log(rng, 1, 4096), "k": 16 * _log(rng, 2, 512), "n": _log(rng, 8, 16384),
                "act": rng.choice(["", "", "silu", "gelu_approx"]), "extra": rng.random() < 0.3}
    kv = rng.choice([1, 2, 4, 8])
    d = rng.choice([32, 64, 80, 96, 128, 256])
    # at most 2^25 values: the largest listed case has 4608 * 72 * 128
    heads = kv * rng.choice([1, 2, 4, 7])
    b = _log(rng, 1, 16)
    top = max(1, min(8192, (1 << 25) // (b * (heads + 2 * kv) * d)))
    return {"op": op, "b": b, "n": _log(rng, 1, top), "heads": heads, "kv": kv, "d": d,
            "rope": rng.choice([d, d, d // 2 // 16 * 16]), "pad": rng.choice([0, 0, 256, 1000]),
            "pairs": rng.choice(["interleaved", "halves"]), "dtype": rng.choice(["bf16", "bf16", "f32"]),
            "positions": rng.random() < 0.5}


# ---------------------------------------------------------------- plain forms
def _exponent_byte(amax):
    """The e8m0 byte of 2^e, e the least integer with amax <= 448 * 2^e (at least -126), from the
    bits of the f32 amax = 1.f * 2^E: E - 8, one more when 1.f > 1.75 = 448 / 256."""
    bits = amax.contiguous().view(torch.int32)
    return ((bits >> 23) - 8 + ((bits & 0x7FFFFF) > 0x600000).to(torch.int32)).clamp(min=1)


def _power(byte):
    """2^(byte - 127) as f32, exactly (bytes 1 .. 254)."""
    return (byte.to(torch.int32) << 23).view(torch.float32)


def _plain_quantize(x):
    """x [M, K] -> q e4m3 [M, K], scales e8m0 [ceil(K / 128), M]."""
    m, k = x.shape
    kb = -(-k // BLOCK)
    g = torch.zeros(m, kb * BLOCK, device=x.device)
    g[:, :k] = x.float()
    g = g.view(m, kb, BLOCK)
    byte = _exponent_byte(g.abs().amax(-1))
    q = (g * _power(254 - byte)[..., None]).to(torch.float8_e4m3fn)
    return q.view(m, kb * BLOCK)[:, :k].contiguous(), byte.t().contiguous().to(torch.uint8).view(torch.float8_e8m0fnu)


def _plain_weight(w):
    """w [N, K] -> q e4m3 [N, K], scales e8m0 [ceil(N / 128), ceil(K / 128)]."""
    n, k = w.shape
    nb, kb = -(-n // BLOCK), -(-k // BLOCK)
    g = torch.zeros(nb * BLOCK, kb * BLOCK, device=w.device)
    g[:n, :k] = w.float()
    g = g.view(nb, BLOCK, kb, BLOCK)
    byte = _exponent_byte(g.abs().amax((1, 3)))
    q = (g * _power(254 - byte)[:, None, :, None]).to(torch.float8_e4m3fn)
    q = q.view(nb * BLOCK, kb * BLOCK)[:n, :k].contiguous()
    return q, byte.to(torch.uint8).view(torch.float8_e8m0fnu)


def _spread_x(xs, m, k):
    return xs.t().repeat_interleave(BLOCK, 1)[:m, :k]


def _spread_w(ws, n, k):
    return ws.repeat_interleave(BLOCK, 0).repeat_interleave(BLOCK, 1)[:n, :k]


def _plain_matmul(s):
    m, k = s["xq"].shape
    n = s["wq"].shape[0]
    x = s["xq"].float() * _spread_x(_power(s["xs"].view(torch.uint8)), m, k)
    w = s["wq"].float() * _spread_w(_power(s["ws"].view(torch.uint8)), n, k)
    y = x @ w.t() + s["bias"].float()
    if s["act"] == "silu":
        y = y / (1.0 + torch.exp(-y))
    elif s["act"] == "gelu_approx":
        y = 0.5 * y * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (y + 0.044715 * y * y * y)))
    if s["gate"] is not None:
        y = s["residual"].float() + s["gate"].float() * y
    return y.to(torch.bfloat16)


def _plain_head(x, w, cos, sin, rope, pairs, eps):
    """x [b, n, h, d] f32, cos / sin [b or 1, n, rope / 2] -> [b, h, n, d]."""
    if w is not None:
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + eps) * w
        c, s = cos[:, :, None, :], sin[:, :, None, :]
        if pairs == "interleaved":
            r = x[..., :rope].unflatten(-1, (rope // 2, 2))
            a, b = r[..., 0], r[..., 1]
            t = torch.stack((a * c - b * s, a * s + b * c), -1).flatten(-2)
        else:
            a, b = x[..., : rope // 2], x[..., rope // 2: rope]
            t = torch.cat((a * c - b * s, a * s + b * c), -1)
        x = torch.cat((t, x[..., rope:]), -1)
    return x.transpose(1, 2)


def _plain_qk(s, up):
    dt = s["q"].dtype
    cos, sin = s["cos"].to(up), s["sin"].to(up)
    if s["positions"] is None:
        n = s["q"].shape[1]
        cos, sin = cos[None, :n], sin[None, :n]
    else:
        cos, sin = cos[s["positions"].long()], sin[s["positions"].long()]
    out = [_plain_head(s[t].to(up), None if w is None else w.to(up), cos, sin, s["rope"], s["pairs"], s["eps"])
           for t, w in (("q", s["qw"]), ("k", s["kw"]), ("v", None))]
    return [o.contiguous() if up == torch.float64 else o.to(dt).contiguous() for o in out]


# ---------------------------------------------------------------- one case
def _outlying(g, *shape):
    """Activations as a transformer block has them: normal, a few channels tens of times larger."""
    x = torch.randn(*shape, device="cuda", generator=g)
    return x * torch.where(torch.rand(shape[-1], device="cuda", generator=g) < 0.01, 30.0, 1.0)


def prepare(case, seed):
    g = torch.Generator("cuda").manual_seed(seed)
    op = case["op"]
    if op == "quantize":
        return {"op": op, "x": _outlying(g, case["m"], case["k"]).to(_DT[case["dtype"]])}
    if op == "weight":
        w = torch.randn(case["n"], case["k"], device="cuda", generator=g) / math.sqrt(case["k"])
        return {"op": op, "w": w.to(_DT[case["dtype"]])}
    if op == "matmul":
        m, k, n = case["m"], case["k"], case["n"]
        xq, xs = _plain_quantize(_outlying(g, m, k))
        wq, ws = _plain_weight(torch.randn(n, k, device="cuda", generator=g) / math.sqrt(k))
        bf = lambda *shape: torch.randn(*shape, device="cuda", generator=g).to(torch.bfloat16)  # noqa: E731
        return {"op": op, "xq": xq, "xs": xs, "wq": wq, "ws": ws, "bias": bf(n), "act": case["act"],
                "gate": bf(n) if case["extra"] else None, "residual": bf(m, n) if case["extra"] else None}
    b, n, h, kv, d, rope = (case[x] for x in ("b", "n", "heads", "kv", "d", "rope"))
    dt = _DT[case["dtype"]]
    qkv = torch.randn(b, n, (h + 2 * kv) * d + case["pad"], device="cuda", generator=g).to(dt)
    # Tables of cos / sin by position; a sequence that decodes reads them at its own place.
    rows = 8192
    angle = torch.arange(rows, device="cuda", dtype=torch.float64)[:, None] * \
        1e4 ** (-torch.arange(rope // 2, device="cuda", dtype=torch.float64) * 2 / max(rope, 1))
    weights = [(1.0 + 0.1 * torch.randn(d, device="cuda", generator=g)).to(dt) for _ in range(2)]
    positions = torch.randint(0, rows, (b, n), device="cuda", generator=g) if case["positions"] else None
    q, k, v = (t.unflatten(-1, (-1, d)) for t in qkv[..., : (h + 2 * kv) * d].split([h * d, kv * d, kv * d], -1))
    return {"op": op, "q": q, "k": k, "v": v, "qw": weights[0], "kw": weights[1], "cos": angle.cos().float(),
            "sin": angle.sin().float(), "rope": rope, "pairs": case["pairs"], "positions": positions, "eps": 1e-6}


def run(state):
    s, op = state, state["op"]
    if own:
        sdq = _sdq()
        if op == "quantize":
            return sdq.fp8_quantize(s["x"])
        if op == "weight":
            return sdq.fp8_quantize_weight(s["w"])
        if op == "matmul":
            return sdq.fp8_matmul(s["xq"], s["xs"], s["wq"], s["ws"], bias=s["bias"], act=s["act"] or None,
                                  gate=s["gate"], residual=s["residual"])
        return sdq.qk_norm_rope(s["q"], s["k"], s["v"], q_weight=s["qw"], k_weight=s["kw"], cos=s["cos"], sin=s["sin"],
                                eps=s["eps"], positions=s["positions"], pairs=s["pairs"])
    if op == "quantize":
        return _plain_quantize(s["x"])
    if op == "weight":
        return _plain_weight(s["w"])
    if op == "matmul":
        return _plain_matmul(s)
    return _plain_qk(s, torch.float32)


def work(case):
    op = case["op"]
    size = 4 if case.get("dtype") == "f32" else 2
    if op == "quantize":
        m, k = case["m"], case["k"]
        return {"bytes": m * k * (size + 1) + m * -(-k // BLOCK), "flops": 0}
    if op == "weight":
        n, k = case["n"], case["k"]
        return {"bytes": n * k * (size + 1) + -(-n // BLOCK) * -(-k // BLOCK), "flops": 0}
    if op == "matmul":
        m, k, n = case["m"], case["k"], case["n"]
        kb = -(-k // BLOCK)
        extra = 2 * n + 2 * m * n if case["extra"] else 0
        return {"bytes": m * k + n * k + m * kb + -(-n // BLOCK) * kb + 2 * n + 2 * m * n + extra, "flops": 2 * m * n * k}
    b, n, h, kv, d, rope = (case[x] for x in ("b", "n", "heads", "kv", "d", "rope"))
    tables = (b * n if case["positions"] else n) * rope * 4 + (8 * b * n if case["positions"] else 0)
    return {"bytes": 2 * b * n * (h + 2 * kv) * d * size + 2 * d * size + tables, "flops": 0}


# ---------------------------------------------------------------- 64 bits
def _round_e4m3(y):
    """The e4m3 number nearest to y (ties to the even one), |y| <= 448, in f64: the step is 2^-3 of
    the power of two below |y|, and 2^-9 under 2^-6."""
    step = torch.exp2(torch.frexp(y).exponent.double().sub(1).clamp(min=-6.0) - 3)
    return torch.round(y / step) * step


def _scale_f64(amax):
    """2^e for the least e >= -126 with amax <= 448 * 2^e: frexp gives amax / 448 = f * 2^p, 1/2 <= f < 1."""
    f, p = torch.frexp(amax / MAX_E4M3)
    e = torch.where(f == 0.5, p - 1, p)
    return torch.exp2(torch.where(amax > 0, e, -126).clamp(min=-126).double())


def _pad(x, *to):
    out = torch.zeros(*to, dtype=torch.float64, device=x.device)
    out[: x.shape[0], : x.shape[1]] = x
    return out


def exact(case, seed):
    s, op = prepare(case, seed), case["op"]
    if op == "quantize":
        m, k = case["m"], case["k"]
        kb = -(-k // BLOCK)
        x = _pad(s["x"].double(), m, kb * BLOCK).unflatten(1, (kb, BLOCK))
        scale = _scale_f64(x.abs().amax(2))
        return _round_e4m3(x / scale[:, :, None]).flatten(1)[:, :k], scale.t()
    if op == "weight":
        n, k = case["n"], case["k"]
        nb, kb = -(-n // BLOCK), -(-k // BLOCK)
        scale = torch.empty(nb, kb, dtype=torch.float64, device="cuda")
        q = torch.empty(n, k, dtype=torch.float64, device="cuda")
        for i in range(nb):
            rows = s["w"][i * BLOCK: (i + 1) * BLOCK].double()
            block = _pad(rows, BLOCK, kb * BLOCK).unflatten(1, (kb, BLOCK))
            scale[i] = _scale_f64(block.abs().amax((0, 2)))
            q[i * BLOCK: (i + 1) * BLOCK] = _round_e4m3(block / scale[i][None, :, None]).flatten(1)[: rows.shape[0], :k]
        return q, scale
    if op == "matmul":
        m, k, n = case["m"], case["k"], case["n"]
        xs, ws = s["xs"].double(), s["ws"].double()
        y = torch.zeros(m, n, dtype=torch.float64, device="cuda")
        of = torch.arange(n, device="cuda") // BLOCK
        for j in range(-(-k // BLOCK)):
            at = slice(j * BLOCK, min(k, (j + 1) * BLOCK))
            y += (s["xq"][:, at].double() * xs[j][:, None]) @ (s["wq"][:, at].double() * ws[of, j][:, None]).t()
        y += s["bias"].double()
        if case["act"] == "silu":
            y = y * torch.sigmoid(y)
        elif case["act"]:
            y = y * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (y + 0.044715 * y ** 3))
        if case["extra"]:
            y = s["residual"].double() + s["gate"].double() * y
        return y
    # Each pair of a head as a complex number times e^(i angle), the norm as a division.
    n = case["n"]
    cos, sin = s["cos"].double(), s["sin"].double()
    turn = torch.complex(cos, sin)
    turn = turn[None, :n] if s["positions"] is None else turn[s["positions"]]
    out, half = [], case["rope"] // 2
    for name, w in (("q", s["qw"]), ("k", s["kw"]), ("v", None)):
        x = s[name].double()
        if w is not None:
            x = x / torch.sqrt((x ** 2).sum(-1, keepdim=True) / case["d"] + s["eps"]) * w.double()
            re, im = (slice(0, 2 * half, 2), slice(1, 2 * half, 2)) if case["pairs"] == "interleaved" \
                else (slice(0, half), slice(half, 2 * half))
            z = torch.complex(x[..., re], x[..., im]) * turn[:, :, None, :]
            x = x.clone()
            x[..., re], x[..., im] = z.real, z.imag
        out.append(x.permute(0, 2, 1, 3).contiguous())
    return out
