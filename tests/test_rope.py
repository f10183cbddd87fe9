"""``rope``, ``qk_norm_rope`` and ``qk_norm_rope_bwd`` against their formulas in float64.

Tolerances count roundings: half a step of the output's type relative to the value, and for what is computed in float32
``C * 2**-24`` of the magnitude of the terms (C: roundings on the way, at worst in the same direction).
"""

import math

import pytest
import torch

import warpy_kernels as wk

FP8 = torch.float8_e4m3fn
U32 = 2.0**-24
EPS = 1e-6


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def axes_of(sections, cycle, pairs):
    if sections is None:
        return [0] * pairs
    if cycle:
        n = len(sections)
        return [j % n if j < n * sections[j % n] else 0 for j in range(pairs)]
    return [a for a, n in enumerate(sections) for _ in range(n)]


def turn_matrix(positions, inv_freq, sections=None, cycle=False):
    """cos and sin in float64, ``[B, 1, N, pairs]``, from ``[B, N]`` or ``[axes, B, N]`` positions."""
    pos = positions.double()
    pos = pos if sections is not None else pos[None]
    axes = axes_of(sections, cycle, inv_freq.shape[0])
    ang = torch.stack([pos[a] * f for a, f in zip(axes, inv_freq.double())], -1)[:, None]
    return ang.cos(), ang.sin()


def pair_indices(pairs, interleaved):
    j = torch.arange(pairs)
    return (2 * j, 2 * j + 1) if interleaved else (j, j + pairs)


def turned(x, cos, sin, interleaved, back=False):
    a, b = pair_indices(cos.shape[-1], interleaved)
    s = -sin if back else sin
    y = x.clone()
    y[..., a], y[..., b] = x[..., a] * cos - x[..., b] * s, x[..., b] * cos + x[..., a] * s
    return y


def pair_size(x, pairs, interleaved):
    """The magnitude of the terms each output is made of."""
    a, b = pair_indices(pairs, interleaved)
    y = x.abs().clone()
    y[..., a] = y[..., b] = x[..., a].abs() + x[..., b].abs()
    return y


def normed(x, w):
    return x * (x.pow(2).mean(-1, keepdim=True) + EPS).rsqrt() * w


def check_forward(got, x, w, cos, sin, interleaved=False, back=False, descale=None):
    """``got`` against the formula on ``x``; 48 roundings: 16 + 4 of the sum of squares (halved by the root), the root,
    three products, angle, cosine and sine, three of the rotation."""
    x, w = x.double(), None if w is None else w.double()
    u = x if w is None else normed(x, w)
    want, terms = turned(u, cos, sin, interleaved, back), pair_size(u, cos.shape[-1], interleaved)
    if descale is not None:
        each = descale.double().repeat_interleave(x.shape[1] // descale.shape[1], 1)[:, :, None, None]
        want, terms = (want / each).clamp(-448, 448), terms / each
        bound = 2.0**-4 * want.abs() + 2.0**-10 + 50 * U32 * terms  # 2^-10: half the step of e4m3's smallest values
    else:
        bound = half_step(got.dtype) * want.abs() + 48 * U32 * terms + torch.finfo(got.dtype).tiny
    err = (got.double() - want).abs()
    assert bool((err <= bound).all()), f"{(err / bound).max().item():.2f} times the bound"


def inputs(B, N, Hq, Hkv, d, dtype, layout, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    if layout == "qkv":
        qkv = torch.randn(B, N, Hq + 2 * Hkv, d, device="cuda", generator=g).to(dtype).transpose(1, 2)
        q, k = qkv[:, :Hq], qkv[:, Hq : Hq + Hkv]
    elif layout == "bnhd":
        q = torch.randn(B, N, Hq, d, device="cuda", generator=g).to(dtype).transpose(1, 2)
        k = torch.randn(B, N, Hkv, d, device="cuda", generator=g).to(dtype).transpose(1, 2)
    elif layout == "odd":  # rows that no 16-byte load can address
        q = torch.randn(B, Hq, N, d + 3, device="cuda", generator=g).to(dtype)[..., 1 : d + 1]
        k = torch.randn(B, Hkv, N, d + 3, device="cuda", generator=g).to(dtype)[..., 2 : d + 2]
    else:
        q = torch.randn(B, Hq, N, d, device="cuda", generator=g).to(dtype)
        k = torch.randn(B, Hkv, N, d, device="cuda", generator=g).to(dtype)
    return q, k, g


def frequencies(pairs, dtype=torch.float32):
    return (10000.0 ** (-torch.arange(pairs, device="cuda", dtype=torch.float64) / pairs)).to(dtype)


def weights(d, g, dtype):
    return tuple((1 + 0.3 * torch.randn(d, device="cuda", generator=g)).to(dtype) for _ in range(2))


CASES = [  # B, N, Hq, Hkv, d, pairs, dtype, layout, interleaved
    (1, 1, 1, 1, 128, 64, torch.bfloat16, "bhnd", False),
    (2, 1, 32, 8, 128, 64, torch.bfloat16, "qkv", False),
    (1, 777, 5, 3, 64, 32, torch.bfloat16, "bnhd", True),
    (3, 129, 7, 1, 128, 32, torch.float16, "qkv", False),
    (2, 33, 8, 2, 80, 40, torch.float16, "bhnd", False),
    (2, 65, 4, 4, 96, 24, torch.float32, "bnhd", True),
    (1, 300, 3, 2, 256, 128, torch.float32, "qkv", False),
    (5, 17, 2, 1, 32, 16, torch.bfloat16, "bhnd", False),
    (1, 1000, 64, 8, 160, 80, torch.bfloat16, "qkv", True),
    (2, 40, 4, 2, 128, 8, torch.bfloat16, "odd", False),
    (1, 40000, 1, 1, 32, 8, torch.float32, "odd", True),
]


@pytest.mark.gpu
@pytest.mark.parametrize("B, N, Hq, Hkv, d, pairs, dtype, layout, interleaved", CASES)
@pytest.mark.parametrize("norm", [False, True])
def test_forward(cuda, B, N, Hq, Hkv, d, pairs, dtype, layout, interleaved, norm):
    q, k, g = inputs(B, N, Hq, Hkv, d, dtype, layout)
    pos = torch.randint(0, 5000, (B, N), device="cuda", generator=g, dtype=torch.int32)
    freq = frequencies(pairs)
    cos, sin = turn_matrix(pos, freq)
    if norm:
        wq, wk_ = weights(d, g, dtype)
        got = wk.qk_norm_rope(q, k, wq, wk_, pos, freq, eps=EPS, interleaved=interleaved)
        check_forward(got[0], q, wq, cos, sin, interleaved)
        check_forward(got[1], k, wk_, cos, sin, interleaved)
        alone, none = wk.qk_norm_rope(q, None, wq, None, pos, freq, eps=EPS, interleaved=interleaved)
    else:
        got = wk.rope(q, k, pos, freq, interleaved=interleaved)
        check_forward(got[0], q, None, cos, sin, interleaved)
        check_forward(got[1], k, None, cos, sin, interleaved)
        check_forward(wk.rope(q, k, pos, freq, interleaved=interleaved, inverse=True)[1], k, None, cos, sin, interleaved, True)
        alone, none = wk.rope(q, None, pos, freq, interleaved=interleaved)
    assert none is None and torch.equal(alone, got[0])


@pytest.mark.gpu
@pytest.mark.parametrize("sections, cycle, pairs", [
    ((16, 24, 24), False, 64), ((24, 20, 20), True, 64), ((0, 32), False, 32), ((32,), False, 32), ((8, 8, 8, 8), True, 32),
    ((40, 12, 12), True, 64), ((1, 2, 3, 34), False, 40), ((12, 0, 4), True, 16),
])
def test_several_axes(cuda, sections, cycle, pairs):
    B, N, d = 2, 50, 128
    q, k, g = inputs(B, N, 4, 2, d, torch.float32, "bnhd")
    pos = torch.randint(-300, 300, (len(sections), B, N), device="cuda", generator=g)
    freq = frequencies(pairs, torch.float64)
    cos, sin = turn_matrix(pos, freq, sections, cycle)
    for x, y in zip((q, k), wk.rope(q, k, pos, freq, sections=sections, cycle=cycle)):
        check_forward(y, x, None, cos, sin)
    # a list is read like a tuple, and positions without a batch go for every item
    y = wk.rope(q, k, pos[:, 0], freq, sections=list(sections), cycle=cycle)[0]
    assert torch.equal(y, wk.rope(q, k, pos[:, :1].expand(-1, B, -1), freq, sections=sections, cycle=cycle)[0])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype, int64", [(torch.int32, False), (torch.int64, True)])
def test_far_positions(cuda, dtype, int64):
    """float32 angles would be whole turns off."""
    far = 2**31 - 1
    pos = torch.tensor([[0, 1, far, -far, 1 << 20, far - 12345] + ([1 << 40] if int64 else [])], device="cuda", dtype=dtype)
    N = pos.shape[1]
    q, k, _ = inputs(1, N, 2, 1, 128, torch.float32, "bhnd")
    freq = frequencies(64)
    cos, sin = turn_matrix(pos, freq)
    got, want = wk.rope(q, k, pos, freq)[0], turned(q.double(), cos, sin, False)
    terms = pair_size(q.double(), 64, False)
    # both sides round pos * f in float64: 2^-53 of up to 2^40 radians, on either side
    bound = 48 * U32 * terms + 4 * 2.0**-53 * pos.abs().double()[:, None, :, None] * terms
    assert bool(((got.double() - want).abs() <= bound).all())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("norm", [False, True])
def test_e4m3_codes(cuda, dtype, norm):
    B, N, Hq, Hkv, d = 2, 70, 6, 3, 128
    q, k, g = inputs(B, N, Hq, Hkv, d, dtype, "qkv")
    pos = torch.arange(N, device="cuda")
    freq = frequencies(64)
    sq, sk = (0.002 + 0.02 * torch.rand(B, Hkv, device="cuda", generator=g) for _ in range(2))  # some values saturate
    cos, sin = turn_matrix(pos.expand(B, N), freq)
    if norm:
        wq, wk_ = weights(d, g, torch.float32)
        got = wk.qk_norm_rope(q, k, wq, wk_, pos, freq, eps=EPS, q_descale=sq, k_descale=sk)
    else:
        wq = wk_ = None
        got = wk.rope(q, k, pos, freq, q_descale=sq, k_descale=sk)
    assert got[0].dtype == FP8 and got[1].dtype == FP8
    check_forward(got[0], q, wq, cos, sin, descale=sq)
    check_forward(got[1], k, wk_, cos, sin, descale=sk)
    out = torch.zeros(B, N + 9, Hkv, d, device="cuda").to(FP8)  # into a cache
    _, there = (wk.qk_norm_rope(q, k, wq, wk_, pos, freq, eps=EPS, q_descale=sq, k_descale=sk, k_out=out[:, 4 : 4 + N].transpose(1, 2))
                if norm else wk.rope(q, k, pos, freq, q_descale=sq, k_descale=sk, k_out=out[:, 4 : 4 + N].transpose(1, 2)))
    assert torch.equal(there.view(torch.uint8), got[1].view(torch.uint8))
    assert not out[:, :4].float().any() and not out[:, 4 + N :].float().any()


@pytest.mark.gpu
def test_outputs_in_place_and_into_a_cache(cuda):
    B, N, Hq, Hkv, d = 2, 45, 4, 2, 64
    q, k, g = inputs(B, N, Hq, Hkv, d, torch.bfloat16, "qkv")
    pos = torch.randint(0, 99, (B, N), device="cuda", generator=g)
    freq = frequencies(32)
    want = wk.rope(q, k, pos, freq)
    cache = torch.full((B, 100, Hkv, d), 7.0, device="cuda", dtype=torch.bfloat16)
    y, z = wk.rope(q, k, pos, freq, k_out=cache[:, 30:75].transpose(1, 2))
    assert torch.equal(y, want[0]) and torch.equal(cache[:, 30:75].transpose(1, 2), want[1])
    assert bool((cache[:, :30] == 7).all()) and bool((cache[:, 75:] == 7).all()) and z.data_ptr() == cache[:, 30:].data_ptr()
    slim = torch.zeros(B, Hq, N, d + 1, device="cuda", dtype=torch.bfloat16)[..., 1:]  # no 16-byte stores there
    assert torch.equal(wk.rope(q, k, pos, freq, q_out=slim)[0], want[0])
    v = q._base if q._base is not None else q
    behind = v.clone()
    y, z = wk.rope(q, k, pos, freq, q_out=q, k_out=k)  # parts of one projection's output, where they are
    assert y is q and torch.equal(q, want[0]) and torch.equal(k, want[1])
    assert torch.equal(v.reshape(B, N, -1, d)[:, :, Hq + Hkv :], behind.reshape(B, N, -1, d)[:, :, Hq + Hkv :])


def grads_of(x, w, dy, cos, sin, interleaved):
    """dx, dw of the formula in float64, and the magnitude of the terms of both."""
    pairs = cos.shape[-1]
    x, w, dy = x.double(), w.double(), dy.double()
    r = (x.pow(2).mean(-1, keepdim=True) + EPS).rsqrt()
    g, big = turned(dy, cos, sin, interleaved, back=True), pair_size(dy, pairs, interleaved)
    h, big_h = g * w, big * w.abs()
    dx = r * (h - x * r * r * (h * x).mean(-1, keepdim=True))
    terms = r * (big_h + x.abs() * r * r * (big_h * x.abs()).mean(-1, keepdim=True))
    return dx, terms, (g * x * r).sum((0, 1, 2)), (big * x.abs() * r).sum((0, 1, 2))


@pytest.mark.gpu
@pytest.mark.parametrize("B, N, Hq, Hkv, d, pairs, dtype, layout, interleaved", CASES)
def test_gradients(cuda, B, N, Hq, Hkv, d, pairs, dtype, layout, interleaved):
    q, k, g = inputs(B, N, Hq, Hkv, d, dtype, layout)
    wt = torch.float32 if N % 2 else dtype
    wq, wk_ = weights(d, g, wt)
    if layout == "odd":  # weights that do not start on 16 bytes
        wq, wk_ = (torch.cat((w[:1], w))[1:] for w in (wq, wk_))
    dq, dk, _ = inputs(B, N, Hq, Hkv, d, dtype, "bhnd" if layout == "qkv" else layout, seed=5)
    pos = torch.randint(0, 5000, (B, N), device="cuda", generator=g, dtype=torch.int32)
    freq = frequencies(pairs)
    cos, sin = turn_matrix(pos, freq)
    got = wk.qk_norm_rope_bwd(dq, dk, q, k, wq, wk_, pos, freq, eps=EPS, interleaved=interleaved)
    for x, w, dy, gx, gw in ((q, wq, dq, got[0], got[2]), (k, wk_, dk, got[1], got[3])):
        dx, terms, dw, dw_terms = grads_of(x, w, dy, cos, sin, interleaved)
        err, bound = (gx.double() - dx).abs(), half_step(dtype) * dx.abs() + 96 * U32 * terms + torch.finfo(dtype).tiny
        assert gx.dtype == dtype and bool((err <= bound).all()), (err / bound).max().item()
        # a thread adds up at most 40000 / 1 / (3 * 148) rows one after the other, then 5 + 8 + 13 + 32 sums
        err, bound = (gw.double() - dw).abs(), half_step(wt) * dw.abs() + (48 + 91 + 58) * U32 * dw_terms
        assert gw.dtype == wt and bool((err <= bound).all()), (err / bound).max().item()
    alone = wk.qk_norm_rope_bwd(dq, None, q, None, wq, None, pos, freq, eps=EPS, interleaved=interleaved)
    assert alone[1] is None and alone[3] is None and torch.equal(alone[0], got[0])
    again = wk.qk_norm_rope_bwd(dq, dk, q, k, wq, wk_, pos, freq, eps=EPS, interleaved=interleaved)
    assert all(torch.equal(a, b) for a, b in zip(got, again)), "the order of the sums must not change"


@pytest.mark.gpu
def test_gradient_against_differences(cuda):
    """Directional derivatives of the formula in float64 by central differences (error of the order of 1e-9)."""
    B, N, Hq, Hkv, d, pairs = 2, 6, 3, 1, 64, 24
    q, _, g = inputs(B, N, Hq, Hkv, d, torch.float32, "bhnd")
    wq = weights(d, g, torch.float32)[0]
    dy = torch.randn(B, Hq, N, d, device="cuda", generator=g)
    pos = torch.randint(0, 3, (3, B, N), device="cuda", generator=g)
    freq, sections = frequencies(pairs), (8, 8, 8)
    cos, sin = turn_matrix(pos, freq, sections, True)
    dq, _, dw, _ = wk.qk_norm_rope_bwd(dy, None, q, None, wq, None, pos, freq, eps=EPS, sections=sections, cycle=True)

    def loss(x, w):
        return (turned(normed(x, w), cos, sin, False) * dy.double()).sum()

    for _ in range(5):
        vx = torch.randn(q.shape, device="cuda", generator=g, dtype=torch.float64)
        vw = torch.randn(d, device="cuda", generator=g, dtype=torch.float64)
        e = 1e-5
        x, w = q.double(), wq.double()
        for got, up, down in ((dq * vx, (x + e * vx, w), (x - e * vx, w)), (dw * vw, (x, w + e * vw), (x, w - e * vw))):
            slope = (loss(*up) - loss(*down)) / (2 * e)
            # 200 float32 roundings at most on every term of the sum
            assert abs(got.double().sum() - slope) <= 200 * U32 * got.abs().double().sum() + 1e-7


@pytest.mark.gpu
def test_rows_do_not_touch_one_another(cuda):
    """NaN and infinity stay in their row (and, through the sum, in the weights' gradient); zero rows have gradients."""
    q, k, g = inputs(1, 9, 4, 2, 128, torch.bfloat16, "bnhd")
    wq, wk_ = weights(128, g, torch.bfloat16)
    pos, freq = torch.arange(9, device="cuda", dtype=torch.int32), frequencies(64)
    clean = wk.qk_norm_rope(q, k, wq, wk_, pos, freq)
    bad = q.clone()
    bad[0, 1, 3, 7], bad[0, 2, 4, 100] = float("nan"), float("inf")
    bad[0, 0, 0] = 0
    y = wk.qk_norm_rope(bad, k, wq, wk_, pos, freq)[0]
    same = torch.ones(1, 4, 9, dtype=torch.bool, device="cuda")
    same[0, 1, 3] = same[0, 2, 4] = same[0, 0, 0] = False
    assert torch.equal(y[same], clean[0][same]) and not y[0, 0, 0].any()
    assert y[0, 1, 3].isnan().all() and y[0, 2, 4].isnan().any()
    dy = torch.randn_like(q)
    dx, _, dw, _ = wk.qk_norm_rope_bwd(dy, torch.zeros_like(k), bad, k, wq, wk_, pos, freq, eps=EPS)
    cos, sin = turn_matrix(pos[None], freq)
    want = grads_of(bad, wq, dy, cos, sin, False)[0]
    assert torch.isfinite(dx[same]).all() and dw.isnan().any()
    err = (dx[0, 0, 0].double() - want[0, 0, 0]).abs()
    assert bool((err <= (half_step(torch.bfloat16) + 96 * U32) * want[0, 0, 0].abs()).all())


@pytest.mark.gpu
def test_lengths_of_zero(cuda):
    freq = frequencies(32)
    for B, N in ((0, 5), (3, 0)):
        q, k = torch.zeros(B, 4, N, 64, device="cuda"), torch.zeros(B, 2, N, 64, device="cuda")
        pos = torch.zeros(B, N, dtype=torch.int32, device="cuda")
        w = torch.ones(64, device="cuda")
        for y, z in (wk.rope(q, k, pos, freq), wk.qk_norm_rope(q, k, w, w, pos, freq)):
            assert y.shape == q.shape and z.shape == k.shape
        dq, dk, dwq, dwk = wk.qk_norm_rope_bwd(q, k, q, k, w, w, pos, freq)
        assert dq.shape == q.shape and dk.shape == k.shape and not dwq.any() and not dwk.any()


@pytest.mark.gpu
def test_streams_and_graphs(cuda):
    B, N, Hq, Hkv, d = 2, 300, 8, 2, 128
    q, k, g = inputs(B, N, Hq, Hkv, d, torch.bfloat16, "qkv")
    wq, wk_ = weights(d, g, torch.bfloat16)
    dq, dk, _ = inputs(B, N, Hq, Hkv, d, torch.bfloat16, "bhnd", seed=3)
    pos, freq = torch.arange(N, device="cuda").expand(B, N), frequencies(64)

    def both():
        return (*wk.qk_norm_rope(q, k, wq, wk_, pos, freq), *wk.qk_norm_rope_bwd(dq, dk, q, k, wq, wk_, pos, freq))

    want = both()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        there = both()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(want, there))
    # two graphs with workspaces of their own, replayed beside one another on new inputs
    graphs, outs = [torch.cuda.CUDAGraph() for _ in range(2)], []
    for graph in graphs:
        with torch.cuda.graph(graph):
            outs.append(both())
    q.mul_(-0.5)
    want = both()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for stream, graph in zip(streams, graphs):
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            for _ in range(3):
                graph.replay()
    torch.cuda.synchronize()
    for got in outs:
        assert all(torch.equal(a, b) for a, b in zip(want, got))


@pytest.mark.gpu
def test_offsets_beyond_32_bits(cuda):
    """Rows more than 2^31 elements into a cache."""
    N, d = 70, 128
    store = torch.empty((1 << 31) + 4 * N * d, device="cuda", dtype=torch.float16)
    far = store.as_strided((2, 1, N, d), (1 << 31, N * d, d, 1), 0)
    q, _, g = inputs(2, N, 1, 1, d, torch.float16, "bhnd")
    pos, freq = torch.arange(N, device="cuda"), frequencies(64)
    want = wk.rope(q, None, pos, freq)[0]
    wk.rope(q, None, pos, freq, q_out=far)
    assert torch.equal(far, want)
    far.copy_(q)
    assert torch.equal(wk.rope(far, None, pos, freq)[0], want)


def test_refusals_before_the_device():
    """What is wrong whatever the GPU: told on the CPU, as ``ValueError``."""
    q = torch.zeros(2, 4, 5, 64)
    k, pos, freq, w = q[:, :2], torch.zeros(2, 5, dtype=torch.int32), torch.ones(32), torch.ones(64)
    bad_q = [q.double(), q[0], torch.zeros(2, 4, 5, 72), torch.zeros(2, 4, 5, 16), torch.zeros(2, 4, 5, 272), torch.zeros(2, 0, 5, 64)]
    for x in bad_q:
        with pytest.raises(ValueError):
            wk.rope(x, None, pos, freq)
        with pytest.raises(ValueError):
            wk.qk_norm_rope(x, None, w, None, pos, freq)
        with pytest.raises(ValueError):
            wk.qk_norm_rope_bwd(x, None, x, None, w, None, pos, freq)
    for x in (k.half(), k[:1], k[:, :, :4], k[..., :32], k[0], k[:, :0]):
        with pytest.raises(ValueError):
            wk.rope(q, x, pos, freq)
    for x in (w[:32], w.double(), None, w[None]):
        with pytest.raises(ValueError):
            wk.qk_norm_rope(q, k, x, w, pos, freq)
        with pytest.raises(ValueError):
            wk.qk_norm_rope(q, k, w, x, pos, freq)
    with pytest.raises(ValueError):
        wk.qk_norm_rope(q, k, w, w.half(), pos, freq)
    with pytest.raises(ValueError):
        wk.qk_norm_rope(q, k, w, w, pos, freq, eps=-1.0)
    for dq, dk in ((q[:1], k), (q.half(), k), (q, None), (q, q)):
        with pytest.raises(ValueError):
            wk.qk_norm_rope_bwd(dq, dk, q, k, w, w, pos, freq)
    if not torch.cuda.is_available():
        for call in (lambda: wk.rope(q, k, pos, freq), lambda: wk.qk_norm_rope(q, k, w, w, pos, freq),
                     lambda: wk.qk_norm_rope_bwd(q, k, q, k, w, w, pos, freq)):
            with pytest.raises(NotImplementedError):
                call()
    assert wk.supports("rope", 100) and wk.supports("qk_norm_rope", 100)


def test_axis_maps():
    from warpy_kernels_b200.rotary import _axis_map

    def read(sections, cycle, pairs):
        words, axes = _axis_map(sections, cycle, pairs)
        assert axes == len(sections)
        return [words[j // 32] >> (2 * (j % 32)) & 3 for j in range(pairs)]

    assert read((2, 3, 3), False, 8) == [0, 0, 1, 1, 1, 2, 2, 2]
    assert read((4, 2, 2), True, 8) == [0, 1, 2, 0, 1, 2, 0, 0]
    assert read((0, 40), False, 40) == [1] * 40
    for sections, cycle in (((4, 5), False), ((9, -1), False), ((1,) * 8, False), ((), False), ((1, 1, 6), True), ((4.0, 4), False)):
        with pytest.raises(ValueError):
            _axis_map(sections, cycle, 8)


@pytest.mark.gpu
def test_refusals(cuda):
    q, k, g = inputs(2, 5, 4, 2, 64, torch.bfloat16, "bhnd")
    pos, freq = torch.zeros(2, 5, dtype=torch.int32, device="cuda"), frequencies(32)
    s = torch.ones(2, 2, device="cuda")
    w = torch.ones(64, device="cuda")
    bad = [
        dict(q=q.cpu(), k=k.cpu(), positions=pos.cpu(), inv_freq=freq.cpu()), dict(k=k.cpu()),
        dict(inv_freq=freq[:31]), dict(inv_freq=freq.half()), dict(inv_freq=torch.ones(40, device="cuda")), dict(inv_freq=freq.cpu()),
        dict(inv_freq=freq[:0]), dict(inv_freq=freq[None]),
        dict(positions=pos[:1, :4]), dict(positions=pos.float()), dict(positions=pos.cpu()), dict(positions=pos[None]),
        dict(positions=pos.short()), dict(sections=(16, 8, 8)), dict(sections=(16, 15), positions=torch.stack((pos, pos))),
        dict(sections=(16, 16, 0), positions=torch.stack((pos, pos))), dict(sections=(2, 30), cycle=True, positions=torch.stack((pos, pos))),
        dict(q_descale=s), dict(k_descale=s), dict(q_descale=s, k_descale=s[:1]), dict(q_descale=s.double(), k_descale=s.double()),
        dict(q_descale=s[:, :1], k_descale=s[:, :1]), dict(q_descale=s.cpu(), k_descale=s.cpu()), dict(q_descale=s[0], k_descale=s[0]),
        dict(q_out=q[:, :2]), dict(q_out=q.float()), dict(q_out=q.cpu()), dict(q_out=q[:, :, :1].expand(-1, -1, 5, -1)),
        dict(k=None, k_out=k), dict(q_out=q[:, :, :4]),
    ]
    for change in bad:
        args = dict(q=q, k=k, positions=pos, inv_freq=freq) | change
        with pytest.raises(ValueError):
            wk.rope(**args)
        with pytest.raises(ValueError):
            ws = w.cpu() if args["q"].device.type == "cpu" else w
            wk.qk_norm_rope(args.pop("q"), args.pop("k"), ws, None if "k" in change and change["k"] is None else ws, **args)
    # an output that lies over its input without being it
    store = torch.zeros(2 * 4 * 6 * 64, device="cuda", dtype=torch.bfloat16)
    x, y = store[: q.numel()].view_as(q), store[64 : 64 + q.numel()].view_as(q)
    with pytest.raises(ValueError):
        wk.rope(x, None, pos, freq, q_out=y)
    with pytest.raises(ValueError):
        wk.rope(q, None, pos, freq, q_out=store.as_strided(q.shape, (320, 64, 64, 1)))
    with pytest.raises(TypeError):
        wk.rope(q, k, pos, freq, no_such_option=1)


@pytest.mark.gpu
def test_a_layer_of_attention(cuda):
    """Projection's output -> norm and rotation -> attention, and back, as a training step runs them, against autograd in
    float64.  The intermediate tensors are bf16: 2^-8 for each of the roundings of q, k, out, P and of the three gradients
    that attention hands on, in the norm over all elements."""
    B, N, Hq, Hkv, d = 2, 200, 4, 2, 128
    g = torch.Generator(device="cuda").manual_seed(7)
    qkv = torch.randn(B, N, Hq + 2 * Hkv, d, device="cuda", generator=g).bfloat16()
    wq, wk_ = weights(d, g, torch.bfloat16)
    dout = torch.randn(B, Hq, N, d, device="cuda", generator=g).bfloat16()
    pos, freq = torch.arange(N, device="cuda"), frequencies(64)
    q, k, v = (x.transpose(1, 2) for x in qkv.split((Hq, Hkv, Hkv), 2))
    qr, kr = wk.qk_norm_rope(q, k, wq, wk_, pos, freq, eps=EPS)
    out, lse, pmax = wk.attn_fwd(qr, kr, v, causal=True)
    dqr, dkr, dv = wk.attn_bwd(qr, kr, v, out, lse, pmax, dout, causal=True)
    dq, dk, dwq, dwk = wk.qk_norm_rope_bwd(dqr, dkr, q, k, wq, wk_, pos, freq, eps=EPS)
    leaves = [x.double().detach().requires_grad_() for x in (q, k, v, wq, wk_)]
    cos, sin = turn_matrix(pos.expand(B, N), freq)
    a, b = (turned_by_product(normed(x, w), cos, sin) for x, w in ((leaves[0], leaves[3]), (leaves[1], leaves[4])))
    scores = a @ b.repeat_interleave(Hq // Hkv, 1).transpose(2, 3) / math.sqrt(d)
    scores = scores.masked_fill(torch.ones(N, N, device="cuda").triu(1).bool(), float("-inf"))
    o = scores.softmax(-1) @ leaves[2].repeat_interleave(Hq // Hkv, 1)
    o.backward(dout.double())
    for got, leaf in zip((dq, dk, dv, dwq, dwk), leaves):
        assert ((got.double() - leaf.grad).norm() / leaf.grad.norm()).item() <= 7 * 2.0**-8
    assert ((out.double() - o).norm() / o.norm()).item() <= 4 * 2.0**-8


def turned_by_product(x, cos, sin):
    pairs = cos.shape[-1]
    a, b = x[..., :pairs], x[..., pairs : 2 * pairs]
    return torch.cat((a * cos - b * sin, b * cos + a * sin, x[..., 2 * pairs :]), -1)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("scale, eps", [(1e14, EPS), (1e17, 0.0), (1e-14, 0.0), (1e-17, 0.0), (1e-14, 1e-30)])
def test_gradients_of_large_and_small_rows(cuda, dtype, scale, eps):
    """Rows whose squares float32 holds, but not the third power of their norm or of its inverse."""
    B, N, H, d, pairs = 2, 9, 3, 64, 32
    g = torch.Generator(device="cuda").manual_seed(11)
    q = (scale * torch.randn(B, H, N, d, device="cuda", generator=g)).to(dtype)
    dy = torch.randn(B, H, N, d, device="cuda", generator=g).to(dtype)
    w = (1 + 0.3 * torch.randn(d, device="cuda", generator=g)).to(dtype)
    pos, freq = torch.arange(N, device="cuda"), frequencies(pairs)
    cos, sin = turn_matrix(pos.expand(B, N), freq)
    x, w64, dy64 = q.double(), w.double(), dy.double()
    r = (x.pow(2).mean(-1, keepdim=True) + eps).rsqrt()
    want, terms = turned(x * r * w64, cos, sin, False), pair_size(x * r * w64, pairs, False)
    got = wk.qk_norm_rope(q, None, w, None, pos, freq, eps=eps)[0]
    assert bool(((got.double() - want).abs() <= half_step(dtype) * want.abs() + 48 * U32 * terms).all())
    gr, big = turned(dy64, cos, sin, False, back=True), pair_size(dy64, pairs, False)
    h, big_h = gr * w64, big * w64.abs()
    dx = r * (h - x * r * (h * x * r).mean(-1, keepdim=True))
    terms = r * (big_h + (x * r).abs() * (big_h * (x * r).abs()).mean(-1, keepdim=True))
    gx, _, gw, _ = wk.qk_norm_rope_bwd(dy, None, q, None, w, None, pos, freq, eps=eps)
    err, bound = (gx.double() - dx).abs(), half_step(dtype) * dx.abs() + 96 * U32 * terms
    assert bool((err <= bound).all()), (err / bound).max().item()
    dw, dw_terms = (gr * x * r).sum((0, 1, 2)), (big * (x * r).abs()).sum((0, 1, 2))
    assert bool(((gw.double() - dw).abs() <= half_step(dtype) * dw.abs() + 200 * U32 * dw_terms).all())


@pytest.mark.gpu
@pytest.mark.parametrize("fp8", [False, True])
def test_outputs_over_one_another(cuda, fp8):
    """An output over the other input or the other output is refused; parts of one tensor that share no byte are not."""
    B, N, Hq, Hkv, d = 2, 33, 4, 2, 64
    q, k, g = inputs(B, N, Hq, Hkv, d, torch.bfloat16, "qkv")
    pos, freq = torch.arange(N, device="cuda"), frequencies(32)
    s = torch.full((B, Hkv), 0.02, device="cuda")
    opts = dict(q_descale=s, k_descale=s) if fp8 else {}
    dtype = FP8 if fp8 else torch.bfloat16
    want = wk.rope(q, k, pos, freq, **opts)
    store = torch.zeros(B, N, Hq + Hkv, d, device="cuda").to(dtype)
    both = store.transpose(1, 2)
    got = wk.rope(q, k, pos, freq, q_out=both[:, Hkv:], k_out=both[:, :Hkv], **opts)  # heads side by side
    for x, y in zip(got, want):
        assert torch.equal(x.view(torch.uint8), y.contiguous().view(torch.uint8))
    before = store.view(torch.uint8).clone()
    w = torch.ones(d, device="cuda")
    odd = lambda x: torch.zeros(B, x.shape[1], N, d + 1, device="cuda").to(x.dtype)[..., 1:].copy_(x)  # left to the Python code
    for a, b in ((q, k), (odd(q), odd(k))):
        bad = [dict(q_out=both[:, :Hq], k_out=both[:, Hq - 1 : Hq - 1 + Hkv]), dict(q_out=both[:, :Hq], k_out=both[:, :Hkv])]
        if not fp8:
            bad += [dict(q_out=b.expand(B, Hkv, N, d).repeat(1, 2, 1, 1)[:, :Hq], k_out=a[:, 1 : 1 + Hkv])]
            if a is q:
                qkv = q._base.transpose(1, 2)  # [B, Hq + 2 Hkv, N, d], k behind q
                bad += [dict(q_out=qkv[:, 1 : 1 + Hq]), dict(q_out=qkv[:, 2 * Hkv :]), dict(q_out=qkv[:, Hkv : Hkv + Hq], k_out=k)]
        for outs in bad:
            with pytest.raises(ValueError, match="overlap"):
                wk.rope(a, b, pos, freq, **opts, **outs)
            with pytest.raises(ValueError, match="overlap"):
                wk.qk_norm_rope(a, b, w, w, pos, freq, **opts, **outs)
    assert torch.equal(store.view(torch.uint8), before)
