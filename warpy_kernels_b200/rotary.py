"""Position rotation of queries and keys, with or without the norm of every head before it, and the gradient of both.

The passes between a layer's projection and ``attn_fwd``: one launch for queries and keys, which can write the e4m3 codes
that the FP8 attention reads, or the keys straight into a cache.  The reference has no such calls (its callers hand
finished ``q`` and ``k`` to ``attn_fwd``, ``warpy_kernels/interface.py:20-64``).
"""

import ctypes

import torch

from . import _lib
from .arch import require
from .utils import apart, overlap, packed_copy

_DTYPES = {torch.bfloat16: _lib.WK_BF16, torch.float16: _lib.WK_F16, torch.float32: _lib.WK_F32}
MAX_AXES = 4


class _RopeArgs(ctypes.Structure):
    _fields_ = [
        *[(name, ctypes.c_void_p) for name in (
            "q", "k", "q_out", "k_out", "q_weight", "k_weight", "q_descale", "k_descale", "positions", "inv_freq",
            "dq_out", "dk_out", "dq_weight", "dk_weight", "workspace")],
        ("workspace_bytes", ctypes.c_int64),
        *[(name, ctypes.c_int64 * 3) for name in (
            "q_strides", "k_strides", "q_out_strides", "k_out_strides", "dq_out_strides", "dk_out_strides",
            "position_strides")],
        ("axis_map", ctypes.c_uint64 * 4),
        *[(name, ctypes.c_int32) for name in (
            "B", "N", "Hq", "Hk", "Hkv", "d", "rot", "dtype", "w_dtype", "position_int64", "inv_freq_f64",
            "interleaved", "inverse")],
        ("eps", ctypes.c_float),
    ]


def _direct(x, unit):
    """Whether the kernels can address ``x``: last stride 1, base and other strides multiples of ``unit`` bytes."""
    size = x.element_size()
    return x.stride(3) == 1 and x.data_ptr() % unit == 0 and all(st * size % unit == 0 for st in x.stride()[:3])


def _check_heads(name, x, like, dtype):
    if x.dim() != 4 or x.dtype != dtype or x.device != like.device:
        raise ValueError(f"{name} must be a [B, H, N, d] {dtype} tensor on {like.device}, got {list(x.shape)} {x.dtype} on {x.device}")
    if x.shape[0] != like.shape[0] or x.shape[2:] != like.shape[2:]:
        raise ValueError(f"{name} must agree with q {list(like.shape)} in all but the heads, got {list(x.shape)}")


def _check_q(q, k):
    if not isinstance(q, torch.Tensor) or q.dim() != 4 or q.dtype not in _DTYPES:
        raise ValueError("q must be a [B, Hq, N, d] bf16, fp16 or float32 tensor")
    d = q.shape[3]
    if d % 16 or not 32 <= d <= 256:
        raise ValueError(f"the head dimension must be a multiple of 16 from 32 to 256, got {d}")
    if q.shape[1] < 1:
        raise ValueError("q has no heads")
    if k is not None:
        _check_heads("k", k, q, q.dtype)
        if k.shape[1] < 1:
            raise ValueError("k has no heads; leave it out instead")


def _check_device(q):
    if not q.is_cuda:
        raise ValueError(f"q must be on a CUDA device, got {q.device}")


def _axis_map(sections, cycle, pairs):
    """Two bits per pair (its position axis) in words of 32 pairs, and the number of axes (0: positions without an axis)."""
    if sections is None:
        return (0, 0, 0, 0), 0
    sections = tuple(sections)
    axes = len(sections)
    if not 1 <= axes <= MAX_AXES or any(not isinstance(n, int) or n < 0 for n in sections) or sum(sections) != pairs:
        raise ValueError(f"sections must be 1 to {MAX_AXES} pair counts that add up to {pairs}, got {sections}")
    if cycle:
        if any(n and a + axes * (n - 1) >= pairs for a, n in enumerate(sections) if a):
            raise ValueError(f"sections {sections} cannot be taken in turn: an axis runs out of pairs")
        of_pair = [j % axes if j < axes * sections[j % axes] else 0 for j in range(pairs)]
    else:
        of_pair = [a for a, n in enumerate(sections) for _ in range(n)]
    words = [0] * 4
    for j, a in enumerate(of_pair):
        words[j // 32] |= a << (2 * (j % 32))
    return tuple(words), axes


def _fill(args, q, k, positions, inv_freq, sections, cycle, interleaved):
    """Checks what all calls share and writes it into the argument block; returns the tensors to keep."""
    B, Hq, N, d = q.shape
    if inv_freq.dim() != 1 or inv_freq.dtype not in (torch.float32, torch.float64) or inv_freq.device != q.device:
        raise ValueError("inv_freq must be a [pairs] float32 or float64 tensor on the device of q")
    pairs = inv_freq.shape[0]
    if pairs % 8 or not 8 <= pairs <= d // 2:
        raise ValueError(f"inv_freq needs a multiple of 8 entries, at most d / 2 = {d // 2}, got {pairs}")
    words, axes = _axis_map(sections, cycle, pairs)
    if positions.dtype not in (torch.int32, torch.int64) or positions.device != q.device:
        raise ValueError("positions must be int32 or int64 on the device of q")
    want = (axes, B, N) if axes else (B, N)
    if positions.shape == want[:-2] + (N,):  # the same for every batch item
        positions = positions.unsqueeze(-2).expand(want)
    if positions.shape != want:
        raise ValueError(f"positions must be {list(want)} or {list(want[:-2] + (N,))}, got {list(positions.shape)}")
    inv_freq = inv_freq.contiguous()
    args.positions, args.inv_freq = positions.data_ptr(), inv_freq.data_ptr()
    args.position_strides = (ctypes.c_int64 * 3)(*(positions.stride() if axes else (0, *positions.stride())))
    args.axis_map = (ctypes.c_uint64 * 4)(*words)
    args.B, args.N, args.Hq, args.Hk, args.d, args.rot = B, N, Hq, 0 if k is None else k.shape[1], d, 2 * pairs
    args.dtype = _DTYPES[q.dtype]
    args.position_int64, args.inv_freq_f64 = int(positions.dtype == torch.int64), int(inv_freq.dtype == torch.float64)
    args.interleaved = int(bool(interleaved))
    return positions, inv_freq


def _put(args, name, x):
    setattr(args, name, x.data_ptr())
    setattr(args, name + "_strides", (ctypes.c_int64 * 3)(*x.stride()[:3]))


def _weight(w):
    """``w`` where the kernels' 16-byte loads can read it."""
    w = w.contiguous()
    return w if w.data_ptr() % 16 == 0 else w.clone()


def _check_weights(q, k, q_weight, k_weight):
    d = q.shape[3]
    for name, w in (("q_weight", q_weight), ("k_weight", k_weight)):
        if w is None and name == "k_weight" and k is None:
            continue
        if not isinstance(w, torch.Tensor) or w.shape != (d,) or w.dtype not in _DTYPES or w.device != q.device:
            raise ValueError(f"{name} must be a [{d}] bf16, fp16 or float32 tensor on the device of q")
    if k is not None and q_weight.dtype != k_weight.dtype:
        raise ValueError("q_weight and k_weight must share a dtype")


def _forward(what, q, k, q_weight, k_weight, positions, inv_freq, eps, sections, cycle, interleaved, inverse, q_out, k_out,
             q_descale, k_descale):
    _check_q(q, k)
    if what == "qk_norm_rope":
        _check_weights(q, k, q_weight, k_weight)
        if not eps >= 0:
            raise ValueError("eps must not be negative")
    require(what, q)
    _check_device(q)
    args = _RopeArgs()
    keep = [_fill(args, q, k, positions, inv_freq, sections, cycle, interleaved)]
    fp8 = q_descale is not None
    if (k is not None and (k_descale is not None) != fp8) or (k is None and k_descale is not None):
        raise ValueError("give both descales, or none")
    dtype = q.dtype
    if fp8:
        dtype = torch.float8_e4m3fn
        B, Hq = q.shape[:2]
        for name, s in (("q_descale", q_descale), ("k_descale", k_descale)):
            if s is None:
                continue
            if s.dim() != 2 or s.dtype != torch.float32 or s.device != q.device or s.shape != q_descale.shape or s.shape[0] != B:
                raise ValueError(f"{name} must be a [B, Hkv] float32 tensor on the device of q")
        hkv = q_descale.shape[1]
        if hkv < 1 or Hq % hkv or (k is not None and k.shape[1] != hkv):
            raise ValueError(f"descales are [B, Hkv] with as many entries as k has heads and Hq a multiple of Hkv, got Hkv = {hkv}")
        q_descale = q_descale.contiguous()
        k_descale = None if k is None else k_descale.contiguous()
        args.q_descale, args.Hkv = q_descale.data_ptr(), hkv
        args.k_descale = None if k is None else k_descale.data_ptr()
        keep += [q_descale, k_descale]
    outs, copies = [], []
    for name, x, out in (("q", q, q_out), ("k", k, k_out)):
        if x is None:
            if out is not None:
                raise ValueError("k_out without k")
            outs.append(None)
            continue
        if out is None:
            out = torch.empty_like(x, dtype=dtype)
        else:
            if out.shape != x.shape or out.dtype != dtype or out.device != x.device or not apart(out):
                raise ValueError(f"{name}_out must be a {dtype} tensor shaped like {name} whose elements do not share memory")
            same = out.data_ptr() == x.data_ptr() and out.stride() == x.stride() and out.dtype == x.dtype
            if not same and overlap(out, x):
                raise ValueError(f"{name}_out may be {name} itself but must not overlap it otherwise")
            for other, y in (("k", k), ("k_out", k_out)) if name == "q" else (("q", q),):
                if y is not None and y.device == out.device and overlap(out, y):
                    raise ValueError(f"{name}_out must not overlap {other}")
        outs.append(out)
        src = x if _direct(x, 16) else packed_copy(x)
        dst = out if _direct(out, 8 if fp8 else 16) else torch.empty(out.shape, dtype=dtype, device=out.device)
        if dst is not out:
            copies.append((out, dst))
        _put(args, name, src)
        _put(args, name + "_out", dst)
        keep += [src, dst]
    if q.numel() == 0:
        return tuple(outs)
    if what == "qk_norm_rope":
        q_weight = _weight(q_weight)
        k_weight = None if k is None else _weight(k_weight)
        args.q_weight, args.w_dtype, args.eps = q_weight.data_ptr(), _DTYPES[q_weight.dtype], float(eps)
        args.k_weight = None if k is None else k_weight.data_ptr()
        keep += [q_weight, k_weight]
    args.inverse = int(bool(inverse))
    lib, host = _lib.lib(), _lib.host()
    _lib.check(host.launch(_lib.address(lib.wk_rope), ctypes.addressof(args), q.device.index), what)
    for out, dst in copies:
        out.copy_(dst)
    return tuple(outs)


def rope(q, k, positions, inv_freq, sections=None, cycle=False, interleaved=False, inverse=False, q_out=None, k_out=None,
         q_descale=None, k_descale=None):
    """Turn queries and keys by their positions, with one or several position axes.

    Pair ``j`` of a head is turned by the angle ``positions[axis of j] * inv_freq[j]``; the angle is reduced in float64,
    so far positions lose nothing.

    Args:
        q: ``[B, Hq, N, d]`` bf16, fp16 or float32, ``d`` a multiple of 16 from 32 to 256. Any strides work if the last one
            is 1, such as the query part of a ``[B, N, Hq + 2 * Hkv, d]`` projection, transposed. Inputs are copied if a
            stride or the base address is not a multiple of 16 bytes.
        k: ``[B, Hkv, N, d]`` of the same dtype, or ``None``.
        positions: ``[B, N]`` int32 or int64, or ``[N]`` for all batch items. With ``sections`` one such tensor per axis:
            ``[axes, B, N]`` or ``[axes, N]``.
        inv_freq: ``[pairs]`` float32 or float64: angle per position of each pair, with whatever scaling a model gives its
            angles (one that multiplies cosine and sine goes into the norm's weights or ``softmax_scale``, where a whole head
            is turned). ``pairs`` is a multiple of 8; the first ``2 * pairs`` elements of a head are turned, the others left.
        sections: How many pairs each position axis turns (time, height, width), up to four, adding up to ``pairs``.
            ``None``: one axis.
        cycle: Pairs take the axes in turn (pair ``j`` axis ``j % axes``) for as long as an axis has pairs left, then the
            first one. ``False``: the first ``sections[0]`` pairs take axis 0, the next ``sections[1]`` axis 1 and so on.
        interleaved: Pair ``j`` is elements ``2 j`` and ``2 j + 1``. ``False``: elements ``j`` and ``j + pairs``.
        inverse: Turn back. That is the gradient: ``rope(dq, dk, ..., inverse=True)``.
        q_out: Output like ``q``, any strides, such as ``q`` itself. ``None`` allocates one with the memory layout of ``q``.
        k_out: The same for ``k``, such as a part of a cache. Outputs must not share a byte with anything but their own input;
            parts of one tensor that lie between one another are fine.
        q_descale: ``[B, Hkv]`` float32: write e4m3 codes of ``q / q_descale``, saturated at 448, which ``attn_fwd`` takes
            with the same descale. ``None``: outputs have the dtype of ``q``.
        k_descale: The same for ``k``. Give both or none.

    Returns:
        ``(q, k)``, turned; the second is ``None`` if ``k`` is.

    Raises:
        ValueError: If a dtype, shape, device or section does not fit, or an output shares a byte with an input or the other
            output without being its own input.
        NotImplementedError: If the GPU is not supported.
    """
    done = _lib.host().rope(q, k, positions, inv_freq, sections, cycle, interleaved, inverse, q_out, k_out, q_descale, k_descale)
    if done is not None:
        return done
    return _forward("rope", q, k, None, None, positions, inv_freq, 0.0, sections, cycle, interleaved, inverse, q_out, k_out,
                    q_descale, k_descale)


def qk_norm_rope(q, k, q_weight, k_weight, positions, inv_freq, eps=1e-6, sections=None, cycle=False, interleaved=False,
                 q_out=None, k_out=None, q_descale=None, k_descale=None):
    """Normalise every head of ``q`` and ``k`` and turn it by its position, in one pass.

    ``u = x * rsqrt(mean(x ** 2) + eps) * weight`` over the ``d`` elements of a head, then the rotation of ``rope``.

    Args:
        q_weight: ``[d]`` bf16, fp16 or float32.
        k_weight: Same dtype; ``None`` if ``k`` is.
        eps: Added to the mean of the squares.
        q, k, positions, inv_freq, sections, cycle, interleaved, q_out, k_out, q_descale, k_descale: As in ``rope``.

    Returns:
        ``(q, k)``, the second ``None`` if ``k`` is.

    Raises:
        ValueError: If a dtype, shape, device or section does not fit, or an output shares a byte with an input or the other
            output without being its own input.
        NotImplementedError: If the GPU is not supported.
    """
    done = _lib.host().qk_norm_rope(q, k, q_weight, k_weight, positions, inv_freq, eps, sections, cycle, interleaved, q_out,
                                    k_out, q_descale, k_descale)
    if done is not None:
        return done
    return _forward("qk_norm_rope", q, k, q_weight, k_weight, positions, inv_freq, eps, sections, cycle, interleaved, False,
                    q_out, k_out, q_descale, k_descale)


def qk_norm_rope_bwd(dq_out, dk_out, q, k, q_weight, k_weight, positions, inv_freq, eps=1e-6, sections=None, cycle=False,
                     interleaved=False):
    """Gradients of ``qk_norm_rope``.

    Args:
        dq_out: Gradient of the first output, shaped and typed like ``q``, such as ``attn_bwd`` returns it.
        dk_out: Gradient of the second one; ``None`` if ``k`` is.
        q, k, q_weight, k_weight, positions, inv_freq, eps, sections, cycle, interleaved: The forward's.

    Returns:
        ``(dq, dk, dq_weight, dk_weight)`` with the dtypes of ``q``, ``k`` and the weights. The weights' gradients are
        summed in float32, always in the same order. The ones of keys are ``None`` if ``k`` is.

    Raises:
        ValueError: If a dtype, shape, device or section does not fit.
        NotImplementedError: If the GPU is not supported.
    """
    done = _lib.host().qk_norm_rope_bwd(dq_out, dk_out, q, k, q_weight, k_weight, positions, inv_freq, eps, sections, cycle,
                                        interleaved)
    if done is not None:
        return done
    _check_q(q, k)
    _check_weights(q, k, q_weight, k_weight)
    if not eps >= 0:
        raise ValueError("eps must not be negative")
    if (k is None) != (dk_out is None):
        raise ValueError("dk_out and k go together")
    for name, x, dy in (("q", q, dq_out), ("k", k, dk_out)):
        if x is not None and (dy.shape != x.shape or dy.dtype != x.dtype or dy.device != x.device):
            raise ValueError(f"d{name}_out must be shaped and typed like {name}, got {list(dy.shape)} {dy.dtype} on {dy.device}")
    require("qk_norm_rope", q)
    _check_device(q)
    args = _RopeArgs()
    keep = [_fill(args, q, k, positions, inv_freq, sections, cycle, interleaved)]
    grads, dws = [], []
    for name, x, dy, w in (("q", q, dq_out, q_weight), ("k", k, dk_out, k_weight)):
        if x is None:
            grads.append(None)
            dws.append(None)
            continue
        src, dsrc = (t if _direct(t, 16) else packed_copy(t) for t in (x, dy))
        w = _weight(w)
        grad = torch.empty_like(x)  # of the memory layout of x, where the kernel can write that
        grads.append(grad if _direct(grad, 16) else torch.empty(x.shape, dtype=x.dtype, device=x.device))
        dws.append(torch.empty_like(w))
        _put(args, name, src)
        _put(args, f"d{name}_out", dsrc)
        _put(args, f"{name}_out", grads[-1])
        setattr(args, f"{name}_weight", w.data_ptr())
        setattr(args, f"d{name}_weight", dws[-1].data_ptr())
        keep += [src, dsrc, w]
    if q.numel() == 0:
        return (*grads, *(None if w is None else w.zero_() for w in dws))
    args.w_dtype, args.eps = _DTYPES[q_weight.dtype], float(eps)
    lib, host = _lib.lib(), _lib.host()
    with torch.cuda.device(q.device):
        args.workspace_bytes = lib.wk_qk_norm_rope_bwd_workspace_bytes(args.d)
    workspace = torch.empty(args.workspace_bytes, dtype=torch.uint8, device=q.device)
    args.workspace = workspace.data_ptr()
    _lib.check(host.launch(_lib.address(lib.wk_qk_norm_rope_bwd), ctypes.addressof(args), q.device.index), "qk_norm_rope_bwd")
    return (*grads, *dws)
