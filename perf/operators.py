"""The operators around attention, as measurable cases: norm and rotation of queries and keys (``qk_norm_rope`` and its
gradient), rotation alone with one or several position axes (``rope``), and attention of a batch over a shared prefix
(``attn_fwd_shared_prefix``).

``own`` says which form ``run`` takes: the plain one in elementary torch operations, or the framework's calls.
"""

import math

import torch

own = False

FP8 = torch.float8_e4m3fn
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
EPS = 1e-6


# ---- cases -------------------------------------------------------------------------------------------------------
def _rope(name, op, dtype, B, N, Hq, Hkv, d, rot, layout, sections="", cycle=False, interleaved=False, out="", wdtype="",
          start=0):
    """``op``: "norm" (norm and rotation), "norm_bwd" (its gradient), "rope" (rotation alone), "rope_bwd" (its gradient).

    ``rot``: how many elements of a head are rotated.  ``sections``: pairs per position axis, "" for one axis.
    ``layout``: "bhnd", "bnhd" or "qkv" (q and k are parts of one projection's output).  ``start``: first position.
    """
    return {"name": name, "kind": "rope", "op": op, "dtype": dtype, "B": B, "N": N, "Hq": Hq, "Hkv": Hkv, "d": d, "rot": rot,
            "layout": layout, "sections": sections, "cycle": cycle, "interleaved": interleaved, "out": out or dtype,
            "wdtype": wdtype or dtype, "start": start}


def _prefix(name, dtype, B, Hq, Hkv, Nq, P, S, d, causal=False, layout="bhnd", lse=False, full=False):
    """``P`` shared keys, then up to ``S`` keys of each sequence's own (``full``: all of them, else a length each)."""
    return {"name": name, "kind": "prefix", "dtype": dtype, "B": B, "Hq": Hq, "Hkv": Hkv, "Nq": Nq, "P": P, "S": S, "d": d,
            "causal": causal, "layout": layout, "lse": lse, "full": full}


def listed():
    return [
        # one generated token of one sequence, far into a context: latency
        _rope("norm_token", "norm", "bf16", 1, 1, 32, 8, 128, 128, "qkv", start=100000),
        # the forward of training at the benchmark's batch: q and k as the projection leaves them
        _rope("norm_train", "norm", "bf16", 4, 4096, 32, 8, 128, 128, "qkv"),
        # a long prompt, written as the e4m3 codes that the FP8 attention reads
        _rope("norm_to_fp8", "norm", "bf16", 1, 32768, 64, 8, 128, 128, "qkv", out="fp8"),
        # its gradient in training: attention's gradients in, gradients of the projection and of both weights out
        _rope("norm_grad", "norm_bwd", "bf16", 4, 4096, 32, 8, 128, 128, "bnhd"),
        # a small model with a ragged length, half of each head rotated, adjacent pairs, float32
        _rope("norm_grad_ragged", "norm_bwd", "fp32", 2, 1000, 4, 2, 64, 32, "bhnd", interleaved=True),
        # video patches: time, height and width, 16-bit floats, heads of 80
        _rope("rope_video", "rope", "fp16", 1, 16385, 16, 16, 80, 80, "qkv", sections="8 16 16"),
        # gradient of a prompt that mixes text and images, axes taken in turn
        _rope("rope_mixed_grad", "rope_bwd", "bf16", 2, 2048, 32, 8, 128, 128, "bnhd", sections="24 20 20", cycle=True),
        # two short sequences of a small model: launch and latency
        _prefix("prefix_short", "bf16", 2, 2, 1, 1, 300, 77, 64, lse=True),
        # decoding 16 sequences that share a prompt, grouped heads
        _prefix("prefix_decode", "bf16", 16, 64, 8, 1, 8192, 1024, 128, layout="bnhd"),
        # a large batch over a long document, FP8 cache: the largest call
        _prefix("prefix_large_fp8", "fp8", 128, 64, 8, 1, 32768, 2048, 128, layout="bnhd"),
        # five drafted tokens checked at once for each of 24 sequences
        _prefix("prefix_draft", "bf16", 24, 32, 8, 5, 4096, 512, 128, causal=True, lse=True),
        # many samples of one prompt without head groups, FP8 cache
        _prefix("prefix_samples_fp8", "fp8", 64, 32, 32, 1, 2048, 300, 128),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _draw_rope(rng):
    op = rng.choice(["norm", "norm", "norm_bwd", "norm_bwd", "rope", "rope_bwd"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    d = rng.choice([32, 64, 80, 96, 128, 128, 128, 160, 256])
    rot = rng.choice([d, d, d, max(16, d // 32 * 16)])
    Hkv = rng.choice([1, 2, 4, 8, 5])
    Hq = Hkv * rng.choice([1, 2, 4, 7, 8])
    most = 0.9e9 / ((3 if op == "norm_bwd" else 2) * (4 if dtype == "fp32" else 2))  # values of the largest listed case's bytes
    N = _log(rng, 1, 40000)
    B = _log(rng, 1, 32)
    N = max(1, min(N, int(most / (B * (Hq + Hkv) * d))))
    sections, cycle = "", False
    if op.startswith("rope") or rng.random() < 0.2:
        h = rot // 2
        if rng.random() < 0.5:
            a = rng.randint(0, h)
            sections = "%d %d" % (a, h - a)
        else:
            a = rng.randint(1, max(1, h // 3))
            sections, cycle = "%d %d %d" % (h - 2 * a, a, a), rng.random() < 0.5
    out = "fp8" if op in ("norm", "rope") and rng.random() < 0.3 else dtype
    return _rope("", op, dtype, B, N, Hq, Hkv, d, rot, rng.choice(["bhnd", "bnhd", "qkv"]), sections, cycle, rng.random() < 0.4,
                 out, rng.choice([dtype, "fp32"]), rng.choice([0, 17, 100000, 1000000]))


def _draw_prefix(rng):
    Hkv, group = rng.choice([1, 2, 4, 8]), rng.choice([1, 2, 4, 7, 8, 16])
    d, Nq = rng.choice([64, 128, 128]), rng.choice([1, 1, 1, 2, 4, 5, 17])
    B, P, S = _log(rng, 1, 128), _log(rng, 40, 32768), _log(rng, 1, 2048)
    while B * Nq * Hkv * group * (P + S) > 64 * 128 * 32768 or B * Hkv * S > 128 * 8 * 2048:
        B, P = max(1, B // 2), max(40, P // 2)
    return _prefix("", rng.choice(["bf16", "fp8"]), B, Hkv * group, Hkv, Nq, P, S, d, Nq > 1 and rng.random() < 0.7,
                   rng.choice(["bhnd", "bnhd"]), rng.random() < 0.5, rng.random() < 0.3)


def draw(rng):
    case = _draw_rope(rng) if rng.random() < 0.5 else _draw_prefix(rng)
    case.pop("name")
    return case


# ---- inputs ------------------------------------------------------------------------------------------------------
def _randn(gen, *shape, dtype=torch.bfloat16):
    return torch.randn(*shape, device="cuda", generator=gen, dtype=dtype)


def _heads(gen, B, H, N, d, layout, dtype):
    """``[B, H, N, d]`` normal values, stored in that order or as ``[B, N, H, d]``."""
    return _randn(gen, B, N, H, d, dtype=dtype).transpose(1, 2) if layout == "bnhd" else _randn(gen, B, H, N, d, dtype=dtype)


def _sections(c):
    return tuple(int(x) for x in c["sections"].split()) or None


def _axes(c):
    """The position axis of every pair."""
    h, sec = c["rot"] // 2, _sections(c) or (c["rot"] // 2,)
    if c["cycle"]:  # the axes in turn for as long as each has pairs left, the first one for the rest
        return [j % len(sec) if j < len(sec) * sec[j % len(sec)] else 0 for j in range(h)]
    return [a for a, n in enumerate(sec) for _ in range(n)]


def _positions(c, gen):
    B, N, start = c["B"], c["N"], c["start"]
    steps = torch.arange(N, device="cuda")
    if not c["sections"]:
        # text: every sequence has its own first position
        first = start + torch.randint(0, 64, (B, 1), device="cuda", generator=gen)
        return (first + steps).to(torch.int32)
    n = len(_sections(c))
    # frames of a grid: time passes slowly, the places in a frame repeat
    side = 24
    axes = [steps // (side * side), steps // side % side, steps % side][-n:]
    shift = torch.randint(0, 64, (n, B, 1), device="cuda", generator=gen)
    return start + shift + torch.stack(axes)[:, None, :]


def _prepare_rope(c, gen):
    B, N, Hq, Hkv, d, dt = c["B"], c["N"], c["Hq"], c["Hkv"], c["d"], DTYPES[c["dtype"]]
    if c["layout"] == "qkv":
        qkv = _randn(gen, B, N, Hq + 2 * Hkv, d, dtype=dt).transpose(1, 2)
        q, k = qkv[:, :Hq], qkv[:, Hq : Hq + Hkv]
    else:
        q, k = _heads(gen, B, Hq, N, d, c["layout"], dt), _heads(gen, B, Hkv, N, d, c["layout"], dt)
    s = {"q": q, "k": k, "positions": _positions(c, gen),
         "inv_freq": 10000.0 ** (-torch.arange(0, c["rot"], 2, device="cuda", dtype=torch.float32) / c["rot"]),
         "axes": torch.tensor(_axes(c), device="cuda"),
         "options": {"sections": _sections(c), "cycle": c["cycle"], "interleaved": c["interleaved"]}}
    if c["op"].startswith("norm"):
        wt = DTYPES[c["wdtype"]]
        s["wq"], s["wk"] = ((1 + 0.2 * _randn(gen, d, dtype=torch.float32)).to(wt) for _ in range(2))
    if c["op"] == "norm_bwd":
        s["dq"], s["dk"] = _randn(gen, B, Hq, N, d, dtype=dt), _randn(gen, B, Hkv, N, d, dtype=dt)
    if c["out"] == "fp8":
        s["sq"], s["sk"] = ((5 + _randn(gen, B, Hkv, dtype=torch.float32).abs()) / 448 for _ in range(2))
    return s


def _to_fp8(x, Hkv):
    """e4m3 codes (in the memory layout of ``x``) and the ``[B, Hkv]`` scale amax / 448 of each batch item and group."""
    B, H = x.shape[:2]
    scale = (x.abs().amax(dim=(2, 3)).view(B, Hkv, H // Hkv).amax(2).float() / 448.0).clamp_min(1e-12)
    return (x / scale.repeat_interleave(H // Hkv, 1).to(x.dtype)[:, :, None, None]).to(FP8), scale


def _prepare_prefix(c, gen):
    B, Hq, Hkv, Nq, P, S, d, lay = (c[x] for x in ("B", "Hq", "Hkv", "Nq", "P", "S", "d", "layout"))
    bf16 = torch.bfloat16
    q = 1.5 * _heads(gen, B, Hq, Nq, d, lay, bf16)
    kp, vp = _heads(gen, 1, Hkv, P, d, lay, bf16), _heads(gen, 1, Hkv, P, d, lay, bf16)
    k, v = _heads(gen, B, Hkv, S, d, lay, bf16), _heads(gen, B, Hkv, S, d, lay, bf16)
    s = {"descales": {}}
    if c["dtype"] == "fp8":
        for name, x in (("q", q), ("k_prefix", kp), ("v_prefix", vp), ("k", k), ("v", v)):
            s[name], s["descales"][name + "_descale"] = _to_fp8(x, Hkv)
    else:
        s.update(q=q, k_prefix=kp, v_prefix=vp, k=k, v=v)
    # lengths between none and the whole room; with a causal mask a sequence holds its queries' own keys at least
    least = min(S, Nq) if c["causal"] else 0
    s["used"] = None if c["full"] else torch.randint(least, S + 1, (B,), device="cuda", generator=gen, dtype=torch.int32)
    return s


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    s = (_prepare_rope if case["kind"] == "rope" else _prepare_prefix)(case, gen)
    s["case"] = case
    return s


# ---- one pass, plain ---------------------------------------------------------------------------------------------
def _angles(s):
    """cos and sin, ``[B, 1, N, pairs]``: the angles in 64 bits."""
    pos = s["positions"]
    pos = pos[None] if pos.dim() == 2 else pos
    ang = pos[s["axes"]].permute(1, 2, 0).double() * s["inv_freq"].double()
    return ang.cos().float()[:, None], ang.sin().float()[:, None]


def _turn(x, cos, sin, rot, interleaved):
    """The first ``rot`` elements of every head turned by the angles, in 32 bits."""
    if interleaved:
        a, b = x[..., 0:rot:2], x[..., 1:rot:2]
        turned = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
    else:
        a, b = x[..., : rot // 2], x[..., rot // 2 : rot]
        turned = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
    return torch.cat((turned, x[..., rot:]), -1)


def _plain_rope(c, s):
    cos, sin = _angles(s)
    outs, grads = [], []
    for x, w, dy, scale in ((s["q"], s.get("wq"), s.get("dq"), s.get("sq")), (s["k"], s.get("wk"), s.get("dk"), s.get("sk"))):
        x32 = x.float()
        if c["op"] == "norm_bwd":
            g = _turn(dy.float(), cos, -sin, c["rot"], c["interleaved"])
            r = torch.rsqrt((x32 * x32).mean(-1, keepdim=True) + EPS)
            grads.append((g * x32 * r).sum((0, 1, 2)).to(w.dtype))
            h = g * w.float()
            outs.append((r * (h - x32 * r * r * (h * x32).mean(-1, keepdim=True))).to(x.dtype))
            continue
        if c["op"] == "norm":
            x32 = x32 * torch.rsqrt((x32 * x32).mean(-1, keepdim=True) + EPS) * w.float()
        y = _turn(x32, cos, -sin if c["op"] == "rope_bwd" else sin, c["rot"], c["interleaved"])
        if scale is None:
            outs.append(y.to(x.dtype))
        else:
            each = scale.repeat_interleave(y.shape[1] // scale.shape[1], 1)[:, :, None, None]
            outs.append((y / each).clamp(-448, 448).to(FP8))
    return (*outs, *grads)


def _plain_prefix(c, s):
    B, Hq, Hkv, Nq, P, S, d = (c[x] for x in ("B", "Hq", "Hkv", "Nq", "P", "S", "d"))
    group, D = Hq // Hkv, s["descales"]
    q, kp, vp, k, v = (s[x].float() for x in ("q", "k_prefix", "v_prefix", "k", "v"))
    if D:
        q = q * D["q_descale"].repeat_interleave(group, 1)[:, :, None, None]
        kp, vp = kp * D["k_prefix_descale"][:, :, None, None], vp * D["v_prefix_descale"][:, :, None, None]
        k, v = k * D["k_descale"][:, :, None, None], v * D["v_descale"][:, :, None, None]
    dev, ninf = q.device, float("-inf")
    used = torch.full((B,), S, device=dev) if s["used"] is None else s["used"].long()
    rows = (q * (1 / math.sqrt(d))).reshape(B, Hkv, group, Nq, d)
    # the prefix: the rows of all sequences that share a KV head at once
    stacked = rows.transpose(0, 1).reshape(Hkv, B * group * Nq, d)
    sp = (stacked @ kp[0].transpose(1, 2)).view(Hkv, B, group, Nq, P)
    ss = (rows.reshape(B, Hkv, group * Nq, d) @ k.transpose(2, 3)).view(B, Hkv, group, Nq, S)
    key, i = torch.arange(S, device=dev), torch.arange(Nq, device=dev)
    last = (used - 1)[:, None].expand(B, Nq)
    if c["causal"]:
        last = torch.minimum(last, i + used[:, None] - Nq)
        seen = torch.arange(P, device=dev) <= (P + i + used[:, None] - Nq)[:, :, None]
        sp = sp.masked_fill(~seen[None, :, None], ninf)
    ss = ss.masked_fill(key > last[:, None, None, :, None], ninf)
    top = torch.maximum(sp.amax(-1).transpose(0, 1), ss.amax(-1) if S else sp.amax(-1).transpose(0, 1))
    ref = top.masked_fill(top == ninf, 0.0)
    sp = torch.exp(sp - ref.transpose(0, 1)[..., None])
    ss = torch.exp(ss - ref[..., None])
    total = sp.sum(-1).transpose(0, 1) + ss.sum(-1)
    o = (sp.view(Hkv, B * group * Nq, P) @ vp[0]).view(Hkv, B, group, Nq, d).transpose(0, 1)
    # what the cache holds behind a sequence's last key takes no part
    v = v.masked_fill((key >= used[:, None])[:, None, :, None], 0.0)
    o = o + (ss.view(B, Hkv, group * Nq, S) @ v).view(B, Hkv, group, Nq, d)
    empty = total == 0
    out = torch.where(empty[..., None], 0.0, o / total[..., None]).reshape(B, Hq, Nq, d).to(torch.bfloat16)
    if not c["lse"]:
        return out
    lse = torch.where(empty, float("inf"), (ref + torch.log(total)) * math.log2(math.e))
    return out, lse.reshape(B, Hq, Nq)


def run(state):
    c, s = state["case"], state
    if not own:
        return _plain_rope(c, s) if c["kind"] == "rope" else _plain_prefix(c, s)
    import warpy_kernels as wk

    if c["kind"] == "prefix":
        out, lse = wk.attn_fwd_shared_prefix(s["q"], s["k_prefix"], s["v_prefix"], s["k"], s["v"], causal=c["causal"],
                                             return_lse=c["lse"], seqused_k=s["used"], **s["descales"])
        return (out, lse) if c["lse"] else out
    if c["op"] == "norm_bwd":
        return wk.qk_norm_rope_bwd(s["dq"], s["dk"], s["q"], s["k"], s["wq"], s["wk"], s["positions"], s["inv_freq"],
                                   eps=EPS, **s["options"])
    if c["op"] == "norm":
        return wk.qk_norm_rope(s["q"], s["k"], s["wq"], s["wk"], s["positions"], s["inv_freq"], eps=EPS,
                               q_descale=s.get("sq"), k_descale=s.get("sk"), **s["options"])
    return wk.rope(s["q"], s["k"], s["positions"], s["inv_freq"], inverse=c["op"] == "rope_bwd", q_descale=s.get("sq"),
                   k_descale=s.get("sk"), **s["options"])


# ---- what a pass cannot do without ---------------------------------------------------------------------------------
def work(case):
    c = case
    if c["kind"] == "rope":
        size = 4 if c["dtype"] == "fp32" else 2
        values = c["B"] * c["N"] * (c["Hq"] + c["Hkv"]) * c["d"]
        each = 3 * size if c["op"] == "norm_bwd" else size + (1 if c["out"] == "fp8" else size)
        positions = c["B"] * c["N"] * (8 * len(_sections(c)) if c["sections"] else 4)
        # norm: squares, their sum, two factors; rotation: three operations an element; about twice that backwards
        return {"bytes": values * each + positions + 2 * c["rot"], "flops": values * {"norm": 7, "norm_bwd": 15}.get(c["op"], 3)}
    B, Hq, Hkv, Nq, P, S, d = (c[x] for x in ("B", "Hq", "Hkv", "Nq", "P", "S", "d"))
    size = 1 if c["dtype"] == "fp8" else 2
    least = min(S, Nq) if c["causal"] else 0
    keys = S if c["full"] else (least + S) / 2  # the mean of the lengths
    rows = B * Hq * Nq
    return {"bytes": 2 * Hkv * d * size * (P + B * keys) + rows * d * (size + 2) + (4 * rows if c["lse"] else 0),
            "flops": 4 * rows * d * (P + keys)}


# ---- the definition in 64 bits -------------------------------------------------------------------------------------
def _exact_rope(c, s):
    rot, h = c["rot"], c["rot"] // 2
    pos = s["positions"].double()
    pos = pos.unsqueeze(0) if pos.dim() == 2 else pos
    # one complex number per pair and token, of modulus 1
    ang = torch.stack([pos[a] * f for a, f in zip(_axes(c), s["inv_freq"].double())], -1)
    z = torch.polar(torch.ones_like(ang), ang)[:, None]

    def turn(x, z):
        first = torch.arange(0, rot, 2) if c["interleaved"] else torch.arange(h)
        second = first + (1 if c["interleaved"] else h)
        y = x.clone()
        w = torch.complex(x[..., first], x[..., second]) * z
        y[..., first], y[..., second] = w.real, w.imag
        return y

    outs, grads = [], []
    for name in "qk":
        x = s[name].double()
        n = (x.pow(2).sum(-1, keepdim=True) / c["d"] + EPS).sqrt()
        if c["op"] == "norm_bwd":
            # y = turn(x / n * w): the chain rule, step by step
            du = turn(s["d" + name].double(), z.conj())
            xn = x / n
            grads.append((du * xn).flatten(0, 2).sum(0))
            dxn = du * s["w" + name].double()
            dn = -(dxn * x).sum(-1, keepdim=True) / n.pow(2)
            outs.append(dxn / n + dn * x / (c["d"] * n))
            continue
        y = x / n * s["w" + name].double() if c["op"] == "norm" else x
        y = turn(y, z.conj() if c["op"] == "rope_bwd" else z)
        if "sq" in s:
            y = (y.unflatten(1, (c["Hkv"], -1)) / s["s" + name].double()[:, :, None, None, None]).flatten(1, 2).clamp(-448, 448)
        outs.append(y)
    return (*outs, *grads)


def _exact_prefix(c, s):
    B, Hq, Hkv, Nq, P, S, d = (c[x] for x in ("B", "Hq", "Hkv", "Nq", "P", "S", "d"))
    if B * Hq * Nq * (P + S) * d > 6e11:
        return None
    D = {n: t.double() for n, t in s["descales"].items()}
    one = torch.ones(B, Hkv, device="cuda", dtype=torch.float64)
    out = torch.zeros(B, Hq, Nq, d, device="cuda", dtype=torch.float64)
    lse = torch.full((B, Hq, Nq), float("inf"), device="cuda", dtype=torch.float64)
    used = [S] * B if s["used"] is None else s["used"].tolist()
    kp = s["k_prefix"][0].double() * D.get("k_prefix_descale", one)[0][:, None, None]
    vp = s["v_prefix"][0].double() * D.get("v_prefix_descale", one)[0][:, None, None]
    for b, n in enumerate(used):  # attention over the concatenated keys of one sequence
        k = torch.cat((kp, s["k"][b, :, :n].double() * D.get("k_descale", one)[b][:, None, None]), 1)
        v = torch.cat((vp, s["v"][b, :, :n].double() * D.get("v_descale", one)[b][:, None, None]), 1)
        q = s["q"][b].double().unflatten(0, (Hkv, -1)) * D.get("q_descale", one)[b][:, None, None, None]
        logits = torch.einsum("hgid,hjd->hgij", q, k) / d**0.5
        if c["causal"]:
            hidden = torch.ones(Nq, P + n, device="cuda", dtype=torch.bool).triu(P + n - Nq + 1)
            logits[..., hidden] = float("-inf")
        z = torch.logsumexp(logits, -1)
        some = z > float("-inf")
        weights = torch.where(some[..., None], torch.exp(logits - z[..., None]), 0.0)
        out[b] = torch.einsum("hgij,hjd->hgid", weights, v).flatten(0, 1)
        lse[b] = torch.where(some, z / math.log(2), float("inf")).flatten(0, 1)
    return (out, lse) if c["lse"] else out


def exact(case, seed):
    s = prepare(case, seed)
    return _exact_rope(case, s) if case["kind"] == "rope" else _exact_prefix(case, s)
