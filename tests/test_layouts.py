"""Tensors that are contiguous to torch but not to the kernels (a base off 16 bytes, dimensions of size 1 with odd strides) are
copied, as the documentation says, and give the same bits."""

import pytest
import torch

import warpy_kernels as wk
from warpy_kernels_b200.utils import overlap, packed_copy

FP8 = torch.float8_e4m3fn


def shifted(x):
    """``x`` one element behind a 16-byte boundary."""
    flat = torch.empty(x.numel() + 16, device=x.device).to(x.dtype)
    y = flat[1 : x.numel() + 1].view(x.shape)
    y.view(torch.uint8).copy_(x.contiguous().view(torch.uint8))
    assert y.is_contiguous() and (y.data_ptr() % 16 or not x.is_cuda)
    return y


def one_strided(x):
    """``[B, H, 1, d]`` whose third dimension has stride 1."""
    y = x.as_strided(x.shape, (*x.contiguous().stride()[:2], 1, 1))
    assert x.shape[2] == 1 and y.is_contiguous()
    return y


def no_batch_stride(x):
    """``[1, H, N, d]`` whose first dimension has stride 3."""
    y = x.as_strided(x.shape, (3, *x.contiguous().stride()[1:]))
    assert x.shape[0] == 1 and y.is_contiguous()
    return y


def same(got, want):
    for x, y in zip(got, want):
        assert (x is None and y is None) or torch.equal(x.view(torch.uint8), y.view(torch.uint8))


def test_a_packed_copy_is_one():
    x = torch.arange(64.0).view(2, 32, 1).transpose(1, 2)
    for y in (shifted(x), one_strided(x[:, None])[:, 0], x.expand(3, 2, 1, 32)[0]):
        z = packed_copy(y)
        assert z.data_ptr() != y.data_ptr() and z.stride() == (32, 32, 1) and torch.equal(z, y)


FORMS = [("shifted", shifted, 2, 7), ("one_strided", one_strided, 2, 1), ("no_batch_stride", no_batch_stride, 1, 7)]


@pytest.mark.gpu
@pytest.mark.parametrize("form, B, N", [f[1:] for f in FORMS], ids=[f[0] for f in FORMS])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_rotation(cuda, form, B, N, dtype):
    g = torch.Generator(device="cuda").manual_seed(0)
    q, k, dq, dk = (torch.randn(B, h, N, 64, device="cuda", generator=g).to(dtype) for h in (4, 2, 4, 2))
    w = torch.randn(64, device="cuda", generator=g).to(dtype)
    pos, freq = torch.arange(N, device="cuda"), torch.rand(32, device="cuda", generator=g)
    want = wk.rope(q, k, pos, freq)
    same(wk.rope(form(q), form(k), pos, freq), want)
    out = torch.zeros_like(q)
    wk.rope(form(q), form(k), pos, freq, q_out=form(out))
    same(wk.qk_norm_rope(form(q), form(k), w, w, pos, freq), wk.qk_norm_rope(q, k, w, w, pos, freq))
    same(wk.qk_norm_rope_bwd(form(dq), form(dk), form(q), form(k), w, w, pos, freq), wk.qk_norm_rope_bwd(dq, dk, q, k, w, w, pos, freq))
    into = form(torch.zeros_like(q))
    got = wk.rope(q, k, pos, freq, q_out=into)
    assert got[0] is into
    same(got, want)


def attention_inputs(B, Nq, Nk, fp8):
    g = torch.Generator(device="cuda").manual_seed(1)
    return [torch.randn(B, h, n, 64, device="cuda", generator=g).to(FP8 if fp8 else torch.bfloat16)
            for h, n in ((4, Nq), (2, Nk), (2, Nk))]


@pytest.mark.gpu
@pytest.mark.parametrize("form, B, N", [f[1:] for f in FORMS], ids=[f[0] for f in FORMS])
@pytest.mark.parametrize("fp8", [False, True])
def test_attention(cuda, form, B, N, fp8):
    for Nq, Nk in ((1, 1),) if N == 1 else ((N, N), (1, 600), (200, 300)):  # the kernels for few rows and the others
        q, k, v = attention_inputs(B, Nq, Nk, fp8)
        ones = [torch.ones(B, 2, device="cuda")] * 3 if fp8 else ()
        want = wk.attn_fwd(q, k, v, *ones)
        same(wk.attn_fwd(form(q), form(k), form(v), *ones), want)
        dout = torch.ones_like(want[0])
        grads = wk.attn_bwd(q, k, v, *want, dout, *ones)
        same(wk.attn_bwd(form(q), form(k), form(v), form(want[0]), *want[1:], form(dout), *ones), grads)


@pytest.mark.gpu
@pytest.mark.parametrize("form, B, N", [f[1:] for f in FORMS], ids=[f[0] for f in FORMS])
@pytest.mark.parametrize("fp8", [False, True])
def test_attention_over_a_shared_prefix(cuda, form, B, N, fp8):
    q, k, v = attention_inputs(B, N, N, fp8)
    kp, vp = (x[:1].clone() for x in (k, v))
    want = wk.attn_fwd_shared_prefix(q, kp, vp, k, v)
    same(wk.attn_fwd_shared_prefix(form(q), form(kp), form(vp), form(k), form(v)), want)
    # a dimension of size 1 without a stride
    flat = [x.as_strided(x.shape, (0, *x.stride()[1:])) for x in (kp, vp)]
    same(wk.attn_fwd_shared_prefix(q, *flat, k, v), want)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("N", [1, 24])
def test_gradients_of_rows_whose_elements_lie_apart(cuda, dtype, N):
    """``[B, H, d, N]`` seen as ``[B, H, N, d]``: read and written, in the forward and in the backward."""
    B, d = 2, 64
    g = torch.Generator(device="cuda").manual_seed(2)
    q, k, dq, dk = (torch.randn(B, h, d, N, device="cuda", generator=g).to(dtype).transpose(2, 3) for h in (4, 2, 4, 2))
    w = torch.randn(d, device="cuda", generator=g).to(dtype)
    pos, freq = torch.arange(N, device="cuda"), torch.rand(32, device="cuda", generator=g)
    flat = [x.clone(memory_format=torch.contiguous_format) for x in (dq, dk, q, k)]
    same((x.contiguous() for x in wk.qk_norm_rope(q, k, w, w, pos, freq)), wk.qk_norm_rope(*flat[2:], w, w, pos, freq))
    got, want = (wk.qk_norm_rope_bwd(*x, w, w, pos, freq) for x in ((dq, dk, q, k), flat))
    assert all(x.shape == y.shape and torch.equal(x, y) for x, y in zip(got, want))


def test_overlap_against_all_addresses():
    """Random shapes and strides, of one and two bytes an element, against the sets of their bytes."""
    g = torch.Generator().manual_seed(5)
    some = lambda values, n: [values[i] for i in torch.randint(len(values), (n,), generator=g).tolist()]
    memory = torch.zeros(2000, dtype=torch.uint8)

    def bytes_of(x):
        at = torch.full((1,), x.data_ptr())
        for st, n in zip(x.stride(), x.shape):
            at = (at[:, None] + st * x.element_size() * torch.arange(n)).flatten()
        return set((at[:, None] + torch.arange(x.element_size())).flatten().tolist())

    met = 0
    for _ in range(1500):
        a, b = (memory.view(t).as_strided(some((1, 2, 3, 4), 4), some((0, 1, 2, 3, 4, 6, 12, 16, 24, 48), 4), some(range(60), 1)[0])
                for t in some((torch.uint8, torch.int16), 2))
        want = bool(bytes_of(a) & bytes_of(b))
        met += want
        assert overlap(a, b) == overlap(b, a) == want
    assert 300 < met < 1200
    x = torch.empty(3, 50, 12, 64).transpose(1, 2)  # a projection's output: its parts share none, its halves in time neither
    assert not overlap(x[:, :4], x[:, 4:8]) and overlap(x[:, :5], x[:, 4:8]) and overlap(x, x)
    assert not overlap(x[:, :, :25], x[:, :, 25:]) and not overlap(x[:0], x) and not overlap(x[..., :32], x[..., 32:])
