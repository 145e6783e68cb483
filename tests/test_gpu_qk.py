"""GPU: queries, keys and values made ready for attention, against the formula in 64 bits.

Tolerance: the norm factor (a sum of d squares, rsqrt within 2 units) is off by at most
(d / 8 + 16) 2^-24 relative, the rotation's two products and their sum by 3 * 2^-24 of
|a| + |b|, plus half a step of the stored type.
"""
from __future__ import annotations

import pytest
import torch

import sdq
from conftest import gpu_available

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not gpu_available(), reason="needs an sm_100 device")]

DT = {"bf16": torch.bfloat16, "f32": torch.float32}
HALF_STEP = {torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}


def normals(seed, *shape):
    g = torch.Generator("cuda").manual_seed(seed)
    return torch.randn(*shape, device="cuda", generator=g)


def tables(rows, rope):
    a = torch.arange(rows, dtype=torch.float64)[:, None] * 1e4 ** (-torch.arange(rope // 2).double() * 2 / max(rope, 1))
    return a.cos().float().cuda(), a.sin().float().cuda()


def head64(x, w, cos, sin, pairs, eps):
    """(value, bound of the sizes entering the last sum) of x [b, n, h, d], cos [b, n, R/2]; [b, h, n, d]."""
    y = x.double()
    if w is not None:
        y = y / (y.pow(2).mean(-1, keepdim=True) + eps).sqrt() * w.double()
    size = y.abs().clone()
    if cos is not None:
        h = cos.shape[-1]
        i = torch.arange(h, device=x.device)
        lo, hi = (2 * i, 2 * i + 1) if pairs == "interleaved" else (i, i + h)
        c, s = cos.double()[:, :, None], sin.double()[:, :, None]
        a, b = y[..., lo], y[..., hi]
        out = y.clone()
        out[..., lo], out[..., hi] = a * c - b * s, a * s + b * c
        size[..., lo] = size[..., hi] = a.abs() + b.abs()
        y = out
    return y.transpose(1, 2), size.transpose(1, 2)


def check(got, x, w, cos, sin, pairs, eps=1e-6):
    want, size = head64(x, w, cos, sin, pairs, eps)
    tol = want.abs() * HALF_STEP[got.dtype] + size * (x.shape[-1] / 8 + 20) * 2.0 ** -24
    bad = ~((got.double() - want).abs() <= tol)
    assert not bad.any(), (int(bad.sum()), got[bad][:4], want[bad][:4])


CASES = [  # b, n, heads, kv heads, d, rope
    (1, 1, 1, 1, 8, 0), (1, 1, 2, 1, 16, 16), (2, 3, 4, 4, 32, 32), (1, 7, 5, 1, 48, 16), (3, 1, 28, 4, 128, 128),
    (1, 129, 24, 24, 128, 128), (2, 33, 14, 2, 80, 80), (1, 65, 8, 8, 96, 48), (1, 40, 7, 1, 256, 256), (2, 300, 1, 1, 64, 32),
    (1, 2, 100, 100, 128, 64),
    # fewer heads than fit a warp: several tokens side by side, the last of them not there
    (3, 37, 1, 1, 32, 32), (2, 5, 3, 1, 16, 16), (1, 9, 9, 1, 64, 64), (5, 3, 2, 2, 8, 0), (1, 41, 33, 1, 32, 16),
    # two and three rounds of a warp's heads
    (3, 37, 4, 2, 96, 48), (1, 21, 7, 1, 64, 64), (2, 9, 2, 1, 256, 256), (1, 17, 6, 3, 128, 64),
]


@pytest.mark.parametrize("pairs", ["interleaved", "halves"])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("b,n,h,kv,d,rope", CASES)
def test_matches_64_bits(b, n, h, kv, d, rope, dtype, pairs):
    """Slices of a fused projection that carries something else behind them, rows by token index."""
    dt = DT[dtype]
    qkv = normals(d + n, b, n, (h + 2 * kv) * d + 24).to(dt)
    q, k, v = (t.unflatten(-1, (-1, d)) for t in qkv[..., :-24].split([h * d, kv * d, kv * d], -1))
    qw, kw = (1 + 0.1 * normals(1, d)).to(dt), (1 + 0.1 * normals(2, d)).to(dt)
    cos, sin = tables(n + 3, rope) if rope else (None, None)
    before = qkv.clone()
    qo, ko, vo = sdq.qk_norm_rope(q, k, v, qw, kw, cos, sin, pairs=pairs)
    assert torch.equal(qkv, before)
    c, s = (cos[None, :n], sin[None, :n]) if rope else (None, None)
    check(qo, q, qw, c, s, pairs)
    check(ko, k, kw, c, s, pairs)
    assert torch.equal(vo, v.transpose(1, 2)) and qo.is_contiguous() and vo.shape == (b, kv, n, d)


@pytest.mark.parametrize("wide", [torch.int32, torch.int64])
@pytest.mark.parametrize("pairs", ["interleaved", "halves"])
def test_positions_and_places_outside_the_tables(pairs, wide):
    b, n, h, kv, d = 3, 5, 4, 2, 64
    q, k, v = normals(1, b, n, h, d), normals(2, b, n, kv, d), normals(3, b, n, kv, d)
    cos, sin = tables(100, d)
    room = torch.tensor([[0, 99, 7, 7, 50, -1], [100, -1, 3, 2, 1, 0], [10, 20, 30, 2 ** 31 - 1, 40, 0]], device="cuda", dtype=wide)
    pos = room[:, :n]                       # rows further apart than n
    qo, ko, vo = sdq.qk_norm_rope(q, k, v, None, None, cos, sin, positions=pos, pairs=pairs)
    out = (pos < 0) | (pos >= 100)
    at = pos.long().clamp(0, 99)
    for got, x in ((qo, q), (ko, k)):
        assert torch.isnan(got.transpose(1, 2)[out]).all()
        fill = got.transpose(1, 2).clone()
        want, _ = head64(x, None, cos[at], sin[at], pairs, 0)
        fill[out] = want.transpose(1, 2)[out].float()
        check(fill.transpose(1, 2), x, None, cos[at], sin[at], pairs)
    assert torch.equal(vo, v.transpose(1, 2))


def test_norm_alone_rotation_alone_and_neither():
    q, k, v = normals(1, 1, 9, 3, 64), normals(2, 1, 9, 1, 64), None
    w = 1 + 0.1 * normals(3, 64)
    cos, sin = tables(9, 32)
    for ww, cc, ss in ((w, None, None), (None, cos, sin), (None, None, None)):
        qo, ko, vo = sdq.qk_norm_rope(q, k, v, ww, None, cc, ss)
        assert vo is None
        c, s = (None, None) if cc is None else (cc[None], ss[None])
        check(qo, q, ww, c, s, "interleaved")
        check(ko, k, None, c, s, "interleaved")


def test_parts_of_a_joint_sequence():
    """Two streams with their own norms written into one [b, h, n1 + n2, d], nothing else touched."""
    b, n1, n2, h, d = 2, 5, 12, 3, 128
    cos, sin = tables(n1 + n2, d)
    joint = [torch.full((b, h, n1 + n2 + 1, d), 9.0, device="cuda", dtype=torch.bfloat16) for _ in range(3)]
    at = 0
    for i, n in enumerate((n1, n2)):
        qkv = normals(40 + i, b, n, 3 * h * d).to(torch.bfloat16)
        q, k, v = (t.unflatten(-1, (h, d)) for t in qkv.chunk(3, -1))
        w = [(1 + 0.1 * normals(50 + 2 * i + j, d)).to(torch.bfloat16) for j in range(2)]
        part = [t[:, :, at:at + n] for t in joint]
        got = sdq.qk_norm_rope(q, k, v, w[0], w[1], cos[at:at + n], sin[at:at + n], out=part)
        assert all(g.data_ptr() == p.data_ptr() for g, p in zip(got, part))
        c, s = cos[None, at:at + n], sin[None, at:at + n]
        check(part[0], q, w[0], c, s, "interleaved")
        check(part[1], k, w[1], c, s, "interleaved")
        assert torch.equal(part[2], v.transpose(1, 2))
        at += n
    assert all((t[:, :, -1] == 9).all() for t in joint)


@pytest.mark.parametrize("pairs", ["interleaved", "halves"])
def test_in_place(pairs):
    b, n, h, d = 2, 17, 6, 64
    q, k = normals(1, b, n, h, d).to(torch.bfloat16), normals(2, b, n, h, d).to(torch.bfloat16)
    w = (1 + 0.1 * normals(3, d)).to(torch.bfloat16)
    cos, sin = tables(n, d)
    want = sdq.qk_norm_rope(q, k, None, w, w, cos, sin, pairs=pairs)
    qt, kt = q.transpose(1, 2), k.transpose(1, 2)
    sdq.qk_norm_rope(q, k, None, w, w, cos, sin, pairs=pairs, out=(qt, kt))
    assert torch.equal(qt, want[0]) and torch.equal(kt, want[1])


def test_rows_of_zeros_infinities_and_nans():
    q = normals(1, 1, 4, 2, 64)
    q[0, 0] = 0
    q[0, 1, 0, 3] = float("inf")
    q[0, 2, 1, 3] = float("nan")
    w = torch.ones(64, device="cuda")
    qo, _, _ = sdq.qk_norm_rope(q, q.clone(), None, w, w)
    want, _ = head64(q, w, None, None, "halves", 1e-6)
    assert torch.equal(torch.isnan(qo), torch.isnan(want)) and (qo[0, :, 0] == 0).all()
    fine = ~torch.isnan(want)
    assert torch.allclose(qo[fine].double(), want[fine], rtol=2.0 ** -18, atol=0)


def test_offsets_past_32_bits():
    """Heads that lie more than 2^31 elements from the base (a slice of a long cache)."""
    d, far = 64, 2 ** 31 + 64
    room = torch.empty(far + 4 * d, device="cuda", dtype=torch.bfloat16)
    q = torch.as_strided(room, (2, 1, 1, d), (far, d, d, 1))
    q.copy_(normals(1, 2, 1, 1, d))
    out = torch.as_strided(room, (2, 1, 1, d), (far, d, d, 1), 2 * d)
    cos, sin = tables(1, d)
    k = normals(2, 2, 1, 1, d).to(torch.bfloat16)
    sdq.qk_norm_rope(q, k, None, None, None, cos, sin, out=(out, torch.empty_like(k)))
    check(out, q, None, cos[None], sin[None], "interleaved")


def test_empty_and_another_stream_and_a_graph():
    e = torch.empty(2, 0, 4, 64, device="cuda")
    assert sdq.qk_norm_rope(e, e, e)[0].shape == (2, 4, 0, 64)
    q, k, v = normals(1, 1, 30, 4, 64), normals(2, 1, 30, 4, 64), normals(3, 1, 30, 4, 64)
    cos, sin = tables(30, 64)
    want = sdq.qk_norm_rope(q, k, v, None, None, cos, sin)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    got = sdq.qk_norm_rope(q, k, v, None, None, cos, sin, stream=s)
    s.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    out = [torch.empty_like(t) for t in want]
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        sdq.qk_norm_rope(q, k, v, None, None, cos, sin, out=out)
    q.copy_(normals(9, 1, 30, 4, 64))
    want = sdq.qk_norm_rope(q, k, v, None, None, cos, sin)
    g.replay()
    assert all(torch.equal(a, b) for a, b in zip(out, want))


@pytest.mark.parametrize("pairs", ["interleaved", "halves"])
def test_the_shortcut_and_ctypes_make_the_same_calls(pairs, monkeypatch):
    from sdq import heads

    q, k, v = normals(1, 2, 9, 4, 64), normals(2, 2, 9, 2, 64), normals(3, 2, 9, 2, 64)
    cos, sin = tables(50, 32)
    w = 1 + 0.1 * normals(4, 64)
    pos = torch.arange(18, device="cuda").view(2, 9)
    place = [torch.empty(2, h, 9, 64, device="cuda") for h in (4, 2, 2)]

    def run():
        return [*sdq.qk_norm_rope(q, k, v, w, w, cos, sin, 1e-5, pos, pairs), *sdq.qk_norm_rope(q, k, None, None, w)[:2],
                *(t.clone() for t in sdq.qk_norm_rope(q, k, v, w, None, cos, sin, positions=pos.int(), pairs=pairs, out=place))]

    quick = run()
    monkeypatch.setattr(heads, "_heads", lambda *args: None)
    assert all(torch.equal(a, b) for a, b in zip(quick, run()))


def test_refusals_of_the_package():
    q, k = normals(1, 1, 4, 2, 64), normals(2, 1, 4, 2, 64)
    cos, sin = tables(4, 64)
    w = torch.ones(64, device="cuda")
    bad = [
        (lambda: sdq.qk_norm_rope(q, k, pairs="quarter"), "pairs must be"),
        (lambda: sdq.qk_norm_rope(q.half(), k.half()), "bf16 or f32"),
        (lambda: sdq.qk_norm_rope(q, k.bfloat16()), "k and its output"),
        (lambda: sdq.qk_norm_rope(q, k[:, :3]), r"k must be \[1, 4"),
        (lambda: sdq.qk_norm_rope(q[0], k), "q must be"),
        (lambda: sdq.qk_norm_rope(q, k, q_weight=w[:32]), "q_weight must hold 64"),
        (lambda: sdq.qk_norm_rope(q, k, k_weight=w.bfloat16()), "k_weight must hold 64"),
        (lambda: sdq.qk_norm_rope(q, k, cos=cos), "cos and sin"),
        (lambda: sdq.qk_norm_rope(q, k, cos=cos, sin=sin[:3]), "sin must be"),
        (lambda: sdq.qk_norm_rope(q, k, cos=cos[:3], sin=sin[:3]), "3 rows for 4 tokens"),
        (lambda: sdq.qk_norm_rope(q, k, positions=torch.zeros(1, 4, device="cuda", dtype=torch.int32)), "positions without"),
        (lambda: sdq.qk_norm_rope(q, k, cos=cos, sin=sin, positions=torch.zeros(1, 4, device="cuda")), "positions must be"),
        (lambda: sdq.qk_norm_rope(q, k, cos=cos, sin=sin, positions=torch.zeros(4, 1, device="cuda", dtype=torch.int32)), "positions must be"),
        (lambda: sdq.qk_norm_rope(q[..., ::2], k[..., ::2]), "contiguous last axis"),
        (lambda: sdq.qk_norm_rope(q[..., :60], k[..., :60]), "head_dim"),
        (lambda: sdq.qk_norm_rope(q, k, out=(q,)), "out must hold 2"),
        (lambda: sdq.qk_norm_rope(q, k, out=(q, k)), "q's output must be"),
        (lambda: sdq.qk_norm_rope(torch.zeros(1, 4, 2, 66, device="cuda")[..., 1:65], k), "aligned"),
    ]
    for call, needle in bad:
        with pytest.raises(sdq.SdqError, match=needle):
            call()
