"""``attn_fwd_shared_prefix`` against attention over the concatenated keys of every sequence in float64.

Tolerances: a probability is rounded to bf16 (2^-8 of its value at most, so 2^-8 of sum p |v|), the output again (2^-8 of its
value); scores are float32 sums of exact products, off by at most 2^-24 of sum |q k| for each of the d additions, which moves
a probability by that, relative, and with the exponent's and the running sums' roundings is far below 2^-10 of sum p |v|.
"""

import math

import pytest
import torch

import warpy_kernels as wk

FP8 = torch.float8_e4m3fn


def quantise(x, Hkv):
    B, H = x.shape[:2]
    s = (x.abs().amax(dim=(2, 3)).view(B, Hkv, H // Hkv).amax(2) / 448 if x.numel() else torch.ones(B, Hkv, device=x.device)).clamp_min(1e-6)
    return (x / s.repeat_interleave(H // Hkv, 1)[:, :, None, None]).to(FP8), s


def make(B, Hq, Hkv, Nq, P, S, d, fp8, seed=0, layout="bhnd", scale=1.5):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def heads(b, H, n):
        if layout == "bnhd":
            return torch.randn(b, n, H, d, device="cuda", generator=g).transpose(1, 2)
        return torch.randn(b, H, n, d, device="cuda", generator=g)

    t = dict(q=scale * heads(B, Hq, Nq), k_prefix=heads(1, Hkv, P), v_prefix=heads(1, Hkv, P), k=heads(B, Hkv, S), v=heads(B, Hkv, S))
    if not fp8:
        return {n: x.bfloat16() for n, x in t.items()}
    out = {}
    for n, x in t.items():
        out[n], out[n + "_descale"] = quantise(x, Hkv)
    return out


def check(t, got, causal=False, seqused_k=None, softmax_scale=None, natural=False):
    """Output and log-sum-exp of every sequence against float64."""
    out, lse = got
    B, Hq, Nq, d = t["q"].shape
    Hkv, P, S = t["k"].shape[1], t["k_prefix"].shape[2], t["k"].shape[2]
    scale = softmax_scale or 1 / math.sqrt(d)
    D = lambda n, b: t[n + "_descale"][b].double()[:, None, None] if n + "_descale" in t else 1.0
    for b in range(B):
        n = S if seqused_k is None else max(0, min(S, int(seqused_k[b])))
        k = torch.cat((t["k_prefix"][0].double() * D("k_prefix", 0), t["k"][b, :, :n].double() * D("k", b)), 1)
        v = torch.cat((t["v_prefix"][0].double() * D("v_prefix", 0), t["v"][b, :, :n].double() * D("v", b)), 1)
        q = (t["q"][b].double().unflatten(0, (Hkv, -1)).flatten(1, 2) * D("q", b)).unflatten(1, (-1, Nq))
        T = P + n
        if T == 0:
            assert not out[b].any() and torch.isposinf(lse[b]).all()
            continue
        s = torch.einsum("hgid,hjd->hgij", q, k) * scale
        slack = torch.einsum("hgid,hjd->hgij", q.abs(), k.abs()) * scale * d * 2.0**-24
        if causal:
            s = s.masked_fill(torch.ones(Nq, T, device="cuda").triu(T - Nq + 1).bool(), float("-inf"))
        m = s.amax(-1, keepdim=True)
        some = (m > float("-inf")).squeeze(-1)
        e = torch.exp(s - m.masked_fill(~some[..., None], 0))
        z = e.sum(-1, keepdim=True)
        p = torch.where(some[..., None], e / z, 0.0)
        want, size = torch.einsum("hgij,hjd->hgid", p, v), torch.einsum("hgij,hjd->hgid", p, v.abs())
        moved = torch.einsum("hgij,hjd->hgid", p * (2 * slack), v.abs())
        err = (out[b].double().unflatten(0, (Hkv, -1)) - want).abs()
        bound = 2.0**-8 * want.abs() + (2.0**-8 + 2.0**-10) * size + moved + 1e-30
        assert bool((err <= bound).all()), f"sequence {b}: {(err / bound).max().item():.2f} times the bound"
        # and on the whole half of that: roundings do not all point one way
        assert err.norm() <= 2.0**-8 * want.norm() + moved.norm() + 1e-30
        x = torch.where(some, m.squeeze(-1) + torch.log(z.squeeze(-1)), float("inf")) * (1 if natural else math.log2(math.e))
        y = lse[b].double().unflatten(0, (Hkv, -1))
        assert torch.equal(torch.isinf(y), ~some)
        # 2^-22 each for exponential and logarithm, the sum's and the last rounding, and what the scores are off by
        assert bool(((y - x).abs()[some] <= (2e-6 + 2.0**-22 * x.abs() + 1.5 * slack.amax(-1))[some]).all())


SHAPES = [  # B, Hq, Hkv, Nq, P, S, d
    (1, 1, 1, 1, 1, 1, 128),
    (2, 2, 1, 1, 300, 77, 64),
    (3, 8, 2, 1, 64, 64, 128),
    (5, 7, 1, 3, 129, 65, 64),
    (17, 16, 8, 1, 1000, 333, 128),
    (40, 32, 4, 1, 777, 200, 128),   # stacked rows of three tiles
    (2, 4, 4, 200, 130, 250, 128),   # a sequence's rows of two tiles
    (64, 8, 8, 2, 2000, 1, 64),
    (1, 16, 1, 1, 20000, 5000, 128),  # few rows, many segments
    (300, 2, 2, 1, 100, 130, 64),
]


@pytest.mark.gpu
@pytest.mark.parametrize("B, Hq, Hkv, Nq, P, S, d", SHAPES)
@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("causal", [False, True])
def test_against_float64(cuda, B, Hq, Hkv, Nq, P, S, d, fp8, causal):
    t = make(B, Hq, Hkv, Nq, P, S, d, fp8, layout="bnhd" if B % 2 else "bhnd")
    check(t, wk.attn_fwd_shared_prefix(**t, causal=causal), causal)
    g = torch.Generator(device="cuda").manual_seed(1)
    used = torch.randint(0, S + 1, (B,), device="cuda", generator=g, dtype=torch.int32)
    used[0] = 0
    check(t, wk.attn_fwd_shared_prefix(**t, causal=causal, seqused_k=used), causal, used)


@pytest.mark.gpu
@pytest.mark.parametrize("B, Hq, Hkv, Nq, P, S, d", [
    (20, 16, 8, 5, 100, 520, 128), (20, 16, 8, 5, 0, 511, 64), (50, 12, 4, 6, 70, 90, 64), (38, 4, 4, 31, 130, 65, 128)])
@pytest.mark.parametrize("fp8", [False, True])
def test_sequences_that_fill_the_gpu(cuda, B, Hq, Hkv, Nq, P, S, d, fp8):
    """Nine rows a sequence and more, where which kernel takes own keys depends on how many and how long they are."""
    t = make(B, Hq, Hkv, Nq, P, S, d, fp8)
    g = torch.Generator(device="cuda").manual_seed(4)
    used = torch.randint(0, S + 1, (B,), device="cuda", generator=g, dtype=torch.int32)
    used[:2] = torch.tensor([0, S], device="cuda", dtype=torch.int32)
    for causal in (False, True):
        check(t, wk.attn_fwd_shared_prefix(**t, causal=causal, seqused_k=used), causal, used)


@pytest.mark.gpu
@pytest.mark.parametrize("fp8", [False, True])
def test_lengths_of_zero(cuda, fp8):
    for P, S in ((0, 100), (100, 0), (0, 0), (0, 1), (1, 0)):
        t = make(3, 4, 2, 2, P, S, 64, fp8)
        for causal in (False, True):
            check(t, wk.attn_fwd_shared_prefix(**t, causal=causal), causal)
    # fewer own keys than queries: with a causal mask the first ones end inside the prefix, or see nothing
    t = make(4, 4, 2, 9, 3, 20, 128, fp8)
    used = torch.tensor([0, 2, 9, 20], device="cuda", dtype=torch.int32)
    got = wk.attn_fwd_shared_prefix(**t, causal=True, seqused_k=used)
    assert not got[0][0, :, :6].any() and torch.isposinf(got[1][0, :, :6]).all()
    check(t, got, True, used)
    # lengths out of range are taken to be the nearest one in it
    used = torch.tensor([-5, 0, 21, 2**30], device="cuda", dtype=torch.int32)
    check(t, wk.attn_fwd_shared_prefix(**t, seqused_k=used), False, used)


@pytest.mark.gpu
@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("d", [64, 128])
def test_what_lies_behind_the_last_key(cuda, fp8, d):
    """NaN and infinities behind a sequence's last key, and neighbours of the output, are left alone."""
    B, Hq, Hkv, Nq, P, S = 5, 8, 2, 2, 200, 300
    t = make(B, Hq, Hkv, Nq, P, S, d, fp8, layout="bnhd")
    used = torch.tensor([0, 1, 63, 64, 170], device="cuda", dtype=torch.int32)
    want = wk.attn_fwd_shared_prefix(**t, seqused_k=used)
    behind = torch.arange(S, device="cuda")[None, :] >= used[:, None]
    for name in "kv":
        codes = t[name].view(torch.uint8 if fp8 else torch.int16)
        bad = (0x7F if fp8 else 0x7FC0) if name == "v" else (0xFF if fp8 else -128)  # -128: 0xff80, minus infinity
        codes.copy_(torch.where(behind[:, None, :, None], torch.tensor(bad, device="cuda").to(codes.dtype), codes))
    room = torch.full((B, Hq, Nq + 2, d + 8), 7.0, device="cuda", dtype=torch.bfloat16)
    out, lse = wk.attn_fwd_shared_prefix(**t, seqused_k=used, out=room[:, :, 1:-1, 4 : d + 4])
    assert torch.equal(out, want[0]) and torch.equal(lse, want[1])
    room[:, :, 1:-1, 4 : d + 4] = 7
    assert bool((room == 7).all())


@pytest.mark.gpu
@pytest.mark.parametrize("fp8", [False, True])
def test_nan_where_it_is_seen(cuda, fp8):
    t = make(2, 4, 2, 1, 100, 50, 128, fp8)
    want = wk.attn_fwd_shared_prefix(**t)[0]
    codes = t["v"].view(torch.uint8 if fp8 else torch.int16)
    codes[1, 0, 7, 3] = 0x7F if fp8 else 0x7FC0
    out = wk.attn_fwd_shared_prefix(**t)[0]
    assert out[1, :2, :, 3].isnan().all()
    out[1, :2, :, 3] = want[1, :2, :, 3]
    assert torch.equal(out, want)
    codes = t["k_prefix"].view(torch.uint8 if fp8 else torch.int16)
    codes[0, 1, 99, 0] = 0x7F if fp8 else 0x7FC0
    out, lse = wk.attn_fwd_shared_prefix(**t)
    assert out[:, 2:].isnan().all() and lse[:, 2:].isnan().all() and not lse[:, :2].isnan().any()


@pytest.mark.gpu
@pytest.mark.parametrize("S", [0, 200])
@pytest.mark.parametrize("Nq", [1, 9, 40])  # own keys by 8 and 16 rows at a time, and by tiles
def test_keys_whose_scores_are_minus_infinity(cuda, Nq, S):
    """They count nothing, also where a segment starts with them; a row that sees nothing else gets 0 and +inf."""
    B, Hq, Hkv, P, d = 3, 4, 2, 300, 128
    t = make(B, Hq, Hkv, Nq, P, S, d, False)
    t["q"].abs_()
    for n, count in (("k_prefix", 170), ("k", 70)):
        t[n][:, :, :count] = float("-inf")
    got = wk.attn_fwd_shared_prefix(**t)
    less = dict(t) | {n: t[n][:, :, 170:] for n in ("k_prefix", "v_prefix")} | {n: t[n][:, :, 70:] for n in "kv"}
    check(less, got)
    t["k_prefix"][:], t["k"][1] = float("-inf"), float("-inf")
    out, lse = wk.attn_fwd_shared_prefix(**t)
    empty = [1] if S else [0, 1, 2]
    assert not out[empty].any() and torch.isposinf(lse[empty]).all()
    assert S == 0 or bool(lse[[0, 2]].isfinite().all())


@pytest.mark.gpu
def test_more_keys_than_are_counted(cuda):
    """No workspace is large enough for them, and the call is refused."""
    from warpy_kernels_b200 import _lib

    size = _lib.lib().wk_attn_fwd_shared_prefix_workspace_bytes
    assert size(1, 1, 1, 1, 1 << 29, 1 << 29, 64) == 0 and size(1, 1, 1, 1, 1 << 29, (1 << 29) - 1, 64) > 0


@pytest.mark.gpu
def test_codes_of_v(cuda):
    """Every e4m3 code of V through the conversion to bf16: one key has all the weight."""
    d = 128
    codes = torch.arange(256, device="cuda", dtype=torch.uint8)
    codes = codes[(codes & 0x7F) != 0x7F]
    v = torch.zeros(1, 1, 128, d, device="cuda", dtype=torch.uint8)
    v[0, 0, 0, :127], v[0, 0, 1, :127] = codes[:127], codes[127:]
    k = torch.zeros(1, 1, 128, d, device="cuda")
    k[0, 0, 0, 0], k[0, 0, 1, 1] = 100, 100
    q = torch.zeros(2, 1, 1, d, device="cuda")
    q[0, 0, 0, 0], q[1, 0, 0, 1] = 100, 100
    empty = torch.zeros(2, 1, 0, d, device="cuda").to(FP8)
    one, two = torch.ones(1, 1, device="cuda"), torch.ones(2, 1, device="cuda")
    out, _ = wk.attn_fwd_shared_prefix(q.to(FP8), k.to(FP8), v.view(FP8), empty, empty, two, two, two, one, one, softmax_scale=1.0)
    assert torch.equal(out[:, 0, 0, :127], torch.stack((codes[:127], codes[127:])).view(FP8).bfloat16())


@pytest.mark.gpu
@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("where", ["prefix", "own"])
def test_scores_far_above_the_first_tile(cuda, fp8, where):
    """Keys that leave the reference of a segment's first tile by more than 2^60, late in the segment."""
    B, Hq, Hkv, Nq, P, S, d = 3, 4, 2, 1, 900, 900, 128
    t = {n: x.float() for n, x in make(B, Hq, Hkv, Nq, P, S, d, False).items()}
    t["q"] = t["q"].abs()
    far = t["k_prefix"][0, :, 850] if where == "prefix" else t["k"][1, :, 777]
    far[:] = 12.0  # about 150 nats for every row
    if fp8:
        out = {}
        for n, x in t.items():
            out[n], out[n + "_descale"] = quantise(x, Hkv)
        t = out
    else:
        t = {n: x.bfloat16() for n, x in t.items()}
    got = wk.attn_fwd_shared_prefix(**t)
    check(t, got)
    # many sequences of one short segment each, beyond what is told apart one by one
    if where == "own":
        t = make(100000, 2, 2, 1, 0, 66, 64, fp8)
        for n in ("k", "q"):
            x = t[n].float()
            if n == "q":
                x = x.abs()
            else:
                x[::7, :, 65] = 100.0
            t[n] = x.to(t[n].dtype)
        whole = wk.attn_fwd_shared_prefix(**t)
        some = torch.cat((torch.arange(0, 30), torch.arange(99970, 100000))).cuda()
        part = {n: (x[some] if x.shape[0] == 100000 else x) for n, x in t.items()}
        check(part, (whole[0][some], whole[1][some]))


@pytest.mark.gpu
@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("rise", [9, 12, 40, 72, -18, -24])
def test_scores_that_rise_within_a_segment(cuda, fp8, rise):
    """Powers of two, so that scores are exact: some keys are 2^rise against the first tile's, within and beyond what its
    reference leaves room for."""
    B, Hq, S, d = 160, 12, 640, 128
    t = make(B, Hq, 1, 1, 130, S, d, fp8)
    for n, value in (("q", 1.0), ("k", 0.0), ("k_prefix", 0.0)):
        x = torch.zeros(t[n].shape, device="cuda")
        x[..., 0] = value
        if n != "q":
            late = slice(64, None) if rise < 0 else slice(x.shape[2] - 20, x.shape[2] - 17)
            x[:, :, late, 0] = rise
        t[n] = x.to(t[n].dtype)
        if fp8:
            t[n + "_descale"] = torch.ones_like(t[n + "_descale"])
    check(t, wk.attn_fwd_shared_prefix(**t, softmax_scale=math.log(2)), softmax_scale=math.log(2))


@pytest.mark.gpu
@pytest.mark.parametrize("fp8", [False, True])
def test_options_and_layouts(cuda, fp8):
    B, Hq, Hkv, Nq, P, S, d = 4, 6, 3, 2, 210, 90, 128
    t = make(B, Hq, Hkv, Nq, P, S, d, fp8)
    out, lse = wk.attn_fwd_shared_prefix(**t, softmax_scale=0.05, lse_natural=True)
    check(t, (out, lse), softmax_scale=0.05, natural=True)
    assert wk.attn_fwd_shared_prefix(**t, return_lse=False)[1] is None
    want = wk.attn_fwd_shared_prefix(**t)
    if fp8:  # without descales they are 1
        bare = {n: x for n, x in t.items() if "descale" not in n}
        ones = {n: torch.ones_like(x) for n, x in t.items() if "descale" in n}
        assert torch.equal(wk.attn_fwd_shared_prefix(**bare)[0], wk.attn_fwd_shared_prefix(**bare, **ones)[0])
    # rows that TMA and 16-byte loads cannot address are copied
    odd = dict(t)
    for n in ("q", "k", "v", "k_prefix", "v_prefix"):
        x = torch.zeros(*t[n].shape[:3], d + 5, device="cuda").to(t[n].dtype)
        x[..., 3 : d + 3] = t[n]
        odd[n] = x[..., 3 : d + 3]
    slim = torch.zeros(B, Hq, Nq, d + 1, device="cuda", dtype=torch.bfloat16)[..., 1:]
    got = wk.attn_fwd_shared_prefix(**odd, out=slim)
    assert got[0] is slim and torch.equal(slim, want[0]) and torch.equal(got[1], want[1])
    # the same keys for all sequences, without memory of their own
    one = {n: (x[:1].expand(B, *x.shape[1:]) if n in ("k", "v", "k_descale", "v_descale") else x) for n, x in t.items()}
    check({n: x.contiguous() for n, x in one.items()}, wk.attn_fwd_shared_prefix(**one))


@pytest.mark.gpu
@pytest.mark.parametrize("fp8", [False, True])
def test_streams_and_graphs(cuda, fp8):
    B = 9
    t = make(B, 8, 2, 1, 1500, 200, 128, fp8)
    used = torch.full((B,), 100, device="cuda", dtype=torch.int32)
    run = lambda: wk.attn_fwd_shared_prefix(**t, seqused_k=used)
    want = run()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        there = [run() for _ in range(5)][-1]
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(there[0], want[0]) and torch.equal(there[1], want[1])
    graphs, outs = [torch.cuda.CUDAGraph() for _ in range(2)], []
    for graph in graphs:
        with torch.cuda.graph(graph):
            outs.append(run())
    used.copy_(torch.arange(B, device="cuda") * 22)  # lengths are read when the graph runs
    want = run()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(3):
        for stream, graph in zip(streams, graphs):
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize()
    for out, lse in outs:
        assert torch.equal(out, want[0]) and torch.equal(lse, want[1])


@pytest.mark.gpu
def test_first_call_of_a_process_inside_a_capture(cuda):
    """Nothing that the library sets up on first use may disturb a capture."""
    import os
    import subprocess
    import sys

    code = """
import torch
import warpy_kernels as wk
t = lambda *s: torch.ones(*s, device="cuda", dtype=torch.bfloat16)
args = t(2, 4, 1, 64), t(1, 2, 70, 64), t(1, 2, 70, 64), t(2, 2, 9, 64), t(2, 2, 9, 64)
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    out, lse = wk.attn_fwd_shared_prefix(*args)
graph.replay()
torch.cuda.synchronize()
assert bool((out == 1).all())
print("replayed")
"""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    res = subprocess.run([sys.executable, "-c", code], cwd=root, capture_output=True, text=True, timeout=300)
    assert res.returncode == 0 and res.stdout.split() == ["replayed"], res.stderr[-800:]


@pytest.mark.gpu
def test_more_sequences_than_are_counted_in_shared_memory(cuda):
    t = make(1500, 2, 1, 1, 70, 20, 64, False)
    g = torch.Generator(device="cuda").manual_seed(2)
    used = torch.randint(0, 21, (1500,), device="cuda", generator=g, dtype=torch.int32)
    check(t, wk.attn_fwd_shared_prefix(**t, seqused_k=used), False, used)


@pytest.mark.gpu
def test_a_long_cache_beyond_32_bits(cuda):
    """Own keys whose offsets pass 2^31 elements."""
    d, S = 128, 40
    store = torch.zeros((1 << 31) + 4 * S * d, device="cuda", dtype=torch.bfloat16)
    t = make(2, 2, 1, 1, 100, S, d, False)
    far = dict(t)
    for i, n in enumerate("kv"):
        far[n] = store.as_strided((2, 1, S, d), (1 << 31, S * d, d, 1), i * S * d)
        far[n].copy_(t[n])
    a, b = wk.attn_fwd_shared_prefix(**t), wk.attn_fwd_shared_prefix(**far)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


@pytest.mark.gpu
@pytest.mark.parametrize("fp8", [False, True])
def test_decoding_steps(cuda, fp8):
    """Norm and rotation write each step's keys into the caches, then the batch attends to prefix and cache, for a few
    tokens in a row; against the same steps on concatenated keys."""
    B, Hq, Hkv, P, S, d = 6, 8, 2, 333, 8, 128
    g = torch.Generator(device="cuda").manual_seed(3)
    randn = lambda *s: torch.randn(*s, device="cuda", generator=g).bfloat16()
    wq, wk_ = 1 + 0.1 * randn(d), 1 + 0.1 * randn(d)
    freq = (10000.0 ** (-torch.arange(64, device="cuda") / 64)).float()
    dtype = FP8 if fp8 else torch.bfloat16
    scales = {n: torch.full((b, Hkv), 0.03, device="cuda") for n, b in (("q", B), ("k", B), ("v", B), ("kp", 1), ("vp", 1))}
    opts = lambda b: dict(q_descale=scales["q"][:b], k_descale=scales["k"][:b]) if fp8 else {}
    dq = lambda x, n: x.float() * (0.03 if fp8 else 1)
    to_v = lambda x: (x.float() / 0.03).to(FP8) if fp8 else x
    # the prompt, once
    _, kp = wk.qk_norm_rope(randn(1, Hq, P, d), randn(1, Hkv, P, d), wq, wk_, torch.arange(P, device="cuda"), freq, **opts(1))
    vp = to_v(randn(1, Hkv, P, d))
    k, v = (torch.zeros(B, Hkv, S, d, device="cuda").to(dtype) for _ in range(2))
    for step in range(S):
        qkv = randn(B, 1, Hq + 2 * Hkv, d).transpose(1, 2)
        pos = torch.full((B, 1), P + step, device="cuda", dtype=torch.int32)
        q, _ = wk.qk_norm_rope(qkv[:, :Hq], qkv[:, Hq : Hq + Hkv], wq, wk_, pos, freq, k_out=k[:, :, step : step + 1], **opts(B))
        v[:, :, step : step + 1] = to_v(qkv[:, Hq + Hkv :])
        used = torch.full((B,), step + 1, device="cuda", dtype=torch.int32)
        t = dict(q=q, k_prefix=kp, v_prefix=vp, k=k, v=v)
        if fp8:
            t |= dict(q_descale=scales["q"], k_descale=scales["k"], v_descale=scales["v"], k_prefix_descale=scales["kp"],
                      v_prefix_descale=scales["vp"])
        got = wk.attn_fwd_shared_prefix(**t, seqused_k=used)
        check(t, got, False, used)
        both = wk.attn_fwd(q, torch.cat((kp.view(torch.uint8).expand(B, *([-1] * 3)), k[:, :, : step + 1].view(torch.uint8)), 2).view(dtype),
                           torch.cat((vp.view(torch.uint8).expand(B, *([-1] * 3)), v[:, :, : step + 1].view(torch.uint8)), 2).view(dtype),
                           *((scales["q"], scales["k"], scales["v"]) if fp8 else ()))
        # two kernels, each within 2^-8 of the row for P and 2^-8 for the output (FP8: P there has 7 bits)
        assert (got[0].float() - both[0].float()).norm() <= 6 * 2.0**-8 * both[0].float().norm()
        assert (got[1] - both[1]).abs().max() <= 1e-4


def bad_calls(q, kp, k, used):
    """Calls that must not reach a kernel."""
    ok = dict(q=q, k_prefix=kp, v_prefix=kp, k=k, v=k)
    for change in (
        dict(q=q.float()), dict(k=k.float()), dict(k_prefix=kp.float(), v_prefix=kp.float()), dict(v=k[:, :, :5]), dict(v_prefix=kp[:, :, :5]),
        dict(k_prefix=kp[0]), dict(k=k[0]), dict(q=q[0]), dict(k_prefix=k, v_prefix=k), dict(k=kp, v=kp), dict(q=q[:, :3]),
        dict(q=q[..., :32], k=k[..., :32], v=k[..., :32], k_prefix=kp[..., :32], v_prefix=kp[..., :32]), dict(q=q[:, :, :0]), dict(q=q[:0], k=k[:0], v=k[:0]),
        dict(k=k[:, :1], v=k[:, :1]), dict(k_prefix=kp[:, :1], v_prefix=kp[:, :1]), dict(softmax_scale=0.0), dict(softmax_scale=-1.0), dict(softmax_scale=float("nan")),
        dict(seqused_k=used.long()), dict(seqused_k=used[:1]), dict(q_descale=used.float()[:, None].expand(-1, 2)),
        dict(out=q[:, :2]), dict(out=q.float()), dict(out=q.transpose(0, 1)),
    ):
        yield ok | change


def test_refusals_on_the_cpu():
    q, kp, k = (torch.zeros(*s, 64, dtype=torch.bfloat16) for s in ((2, 4, 1), (1, 2, 10), (2, 2, 6)))
    used = torch.ones(2, dtype=torch.int32)
    for call in bad_calls(q, kp, k, used):
        with pytest.raises((ValueError, NotImplementedError)):
            wk.attn_fwd_shared_prefix(**call)
    for x in (q.float(), q.half()):
        with pytest.raises(ValueError):
            wk.attn_fwd_shared_prefix(x, kp, kp, k, k)
    assert wk.supports("attn_fwd_shared_prefix", 100)
    from warpy_kernels_b200 import _lib

    assert _lib.lib().wk_attn_fwd_shared_prefix_workspace_bytes(2, 3, 2, 1, 10, 10, 64) == 0


@pytest.mark.gpu
def test_refusals(cuda):
    q, kp, k = (torch.zeros(*s, 64, device="cuda", dtype=torch.bfloat16) for s in ((2, 4, 1), (1, 2, 10), (2, 2, 6)))
    used = torch.ones(2, dtype=torch.int32, device="cuda")
    for call in bad_calls(q, kp, k, used):
        with pytest.raises(ValueError):
            wk.attn_fwd_shared_prefix(**call)
    for change in (dict(q=q.cpu()), dict(k=k.cpu(), v=k.cpu()), dict(v_prefix=kp.cpu()), dict(seqused_k=used.cpu()), dict(out=q.cpu())):
        with pytest.raises(ValueError):
            wk.attn_fwd_shared_prefix(**(dict(q=q, k_prefix=kp, v_prefix=kp, k=k, v=k) | change))
    q8, kp8, k8 = q.to(FP8), kp.to(FP8), k.to(FP8)
    for change in (dict(k_prefix_descale=torch.ones(2, 2, device="cuda")), dict(q_descale=torch.ones(2, 4, device="cuda")), dict(v_descale=torch.ones(2, 2))):
        with pytest.raises(ValueError):
            wk.attn_fwd_shared_prefix(q8, kp8, kp8, k8, k8, **change)
    with pytest.raises(TypeError):
        wk.attn_fwd_shared_prefix(q, kp, kp, k, k, no_such_option=1)


@pytest.mark.gpu
@pytest.mark.parametrize("Nq", [1, 9, 40])
def test_the_output_in_place_of_the_queries(cuda, Nq):
    """``out`` may be ``q``; anything else that it shares a byte with is refused, and so is one that overlaps itself."""
    B, Hq, Hkv, P, S, d = 3, 8, 2, 700, 300, 128
    t = make(B, Hq, Hkv, Nq, P, S, d, False, layout="bnhd")
    want = wk.attn_fwd_shared_prefix(**t)
    room = torch.zeros(B, Nq + 1, Hq + 2, d + 16, device="cuda", dtype=torch.bfloat16).transpose(1, 2)
    inside = dict(t) | dict(q=room[:, 1:-1, :Nq, :d].copy_(t["q"]))
    for call in (inside, dict(t)):
        got = wk.attn_fwd_shared_prefix(**call, out=call["q"])
        assert got[0] is call["q"] and torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    q = room[:, 1:-1, :Nq, :d].copy_(want[0])
    t["q"] = q
    store = torch.zeros(B * Hq * (Nq + 1) * d + 64, device="cuda", dtype=torch.bfloat16)
    memory = dict(q=q, k=t["k"], v=t["v"], k_prefix=t["k_prefix"], v_prefix=t["v_prefix"])
    for name, x in memory.items():
        base = x._base if x._base is not None else x
        flat = base.as_strided((base.untyped_storage().nbytes() // 2,), (1,), 0)
        if flat.numel() < B * Hq * Nq * d + 16:
            continue
        for out in (flat[8 : 8 + B * Hq * Nq * d].view(B, Hq, Nq, d), flat[4 : 4 + B * Hq * Nq * d].view(B, Nq, Hq, d).transpose(1, 2)):
            with pytest.raises(ValueError, match="overlap " + name):
                wk.attn_fwd_shared_prefix(**t, out=out)
    for out in (store.as_strided((B, Hq, Nq, d), (64, 4, d * Hq, 1)), store[:d].expand(B, Hq, Nq, d)):
        with pytest.raises(ValueError, match="share memory"):
            wk.attn_fwd_shared_prefix(**t, out=out)
    between = room[:, 1:-1, 1:, :d]  # tokens one behind the queries': over them, unless there is but one
    if Nq == 1:
        assert torch.equal(wk.attn_fwd_shared_prefix(**t, out=between)[0], wk.attn_fwd_shared_prefix(**t)[0])
    else:
        with pytest.raises(ValueError, match="overlap q"):
            wk.attn_fwd_shared_prefix(**t, out=between)
    t8 = make(B, Hq, Hkv, Nq, P, S, d, True)
    wide = torch.zeros(B, Hq, Nq, 2 * d, device="cuda", dtype=torch.uint8)
    t8["q"] = wide.view(FP8)[..., :d].copy_(t8["q"])
    with pytest.raises(ValueError, match="overlap q"):
        wk.attn_fwd_shared_prefix(**t8, out=wide.view(torch.bfloat16))


@pytest.mark.gpu
@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("Nq", [1, 12])
def test_repeats_itself_beside_other_work(cuda, fp8, Nq):
    """Rings that are refilled while they are read: the same bits every time, also while another stream keeps the memory busy."""
    t = make(7, 8, 8, Nq, 300, 3000, 128, fp8)
    want = wk.attn_fwd_shared_prefix(**t)
    check(t, want)
    side, copy = torch.cuda.Stream(), torch.empty(2, 1 << 28, device="cuda", dtype=torch.uint8)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(20):
            copy[0].copy_(copy[1])
    got = [wk.attn_fwd_shared_prefix(**t) for _ in range(40)]
    torch.cuda.synchronize()
    for out, lse in got:
        assert torch.equal(out, want[0]) and torch.equal(lse, want[1])


@pytest.mark.gpu
@pytest.mark.parametrize("fp8, Nq, P, S", [
    (True, 1, 600, 0), (True, 1, 0, 600), (True, 12, 0, 600), (True, 40, 0, 600), (True, 1, 6000, 90), (False, 1, 600, 0),
    (False, 1, 0, 600), (False, 40, 0, 600)])
@pytest.mark.parametrize("d", [64, 128])
def test_bits_of_the_probabilities(cuda, fp8, Nq, P, S, d):
    """Two thirds of the keys have one and the same probability against the others', (1 + 2^-8 + 2^-12) / 2, and values of the
    other sign, so that the sums nearly cancel and what its rounding leaves is all there is to see: 2^-11 of sum p |v| at most
    in f16 (FP8 inputs), 2^-8 in bf16, which here would be off by 2^-9.  Beside that the exponential (2^-21), one float32
    addition (2^-23) for every 16 keys, and the output's rounding."""
    B, Hq, Hkv = 3, 2, 1
    dtype = FP8 if fp8 else torch.bfloat16
    x = (1 + 2.0**-8 + 2.0**-12) / 2
    q = torch.zeros(B, Hq, Nq, d, device="cuda")
    q[..., 0] = 1
    t = dict(q=q)
    for b, n, names in ((1, P, ("k_prefix", "v_prefix")), (B, S, ("k", "v"))):
        small = (torch.arange(n, device="cuda") % 3 != 0)[None, None, :, None].expand(b, Hkv, n, d).float()
        t[names[0]], t[names[1]] = -small * (torch.arange(d, device="cuda") == 0), 1 - 2 * small
    t = {n: y.to(dtype) for n, y in t.items()}
    out, _ = wk.attn_fwd_shared_prefix(**t, softmax_scale=-math.log(x))
    T = P + S
    many = sum(int((torch.arange(n) % 3 != 0).sum()) for n in (P, S))
    want = ((T - many) - many * x) / ((T - many) + many * x)
    err = (out.double() - want).abs().max().item()
    assert err <= 2.0**-8 * abs(want) + (2.0**-11 if fp8 else 2.0**-8) + 2.0**-21 + T / 16 * 2.0**-23  # sum p |v| is 1


@pytest.mark.gpu
@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("B, Hq, Hkv, Nq, P, S, d", [(3, 4, 2, 512, 700, 512, 128), (2, 2, 1, 777, 130, 900, 64), (1, 3, 3, 300, 0, 300, 128)])
def test_prompts_behind_a_prefix(cuda, fp8, B, Hq, Hkv, Nq, P, S, d):
    """Hundreds of queries a sequence, most of whose tiles the causal mask cuts."""
    t = make(B, Hq, Hkv, Nq, P, S, d, fp8, layout="bnhd")
    check(t, wk.attn_fwd_shared_prefix(**t, causal=True), True)
    used = torch.tensor([S, Nq // 2, 1][:B], device="cuda", dtype=torch.int32)  # and sequences shorter than their queries
    check(t, wk.attn_fwd_shared_prefix(**t, causal=True, seqused_k=used), True, used)
