"""Attention over a prefix of keys that all sequences of a batch share, and each sequence's own keys behind it.

The reference attends sequence by sequence (``warpy_kernels/attn/fwd_api.py:141-548``); layouts, descales, masks and the
meaning of ``lse`` are those of ``attn_fwd``.
"""

import ctypes
import math

import torch

from .. import _lib
from ..arch import require
from ..utils import apart, cached_tensor, check_descale, overlap, packed_copy
from .fwd_api import _check_qkv, _kernel_view


class _PrefixArgs(ctypes.Structure):
    _fields_ = [
        *[(name, ctypes.c_void_p) for name in (
            "q", "k_prefix", "v_prefix", "k", "v", "out", "lse", "q_descale", "k_descale", "v_descale", "k_prefix_descale",
            "v_prefix_descale", "seqused_k", "workspace")],
        ("workspace_bytes", ctypes.c_int64),
        *[(name + "_strides", ctypes.c_int64 * 3) for name in ("q", "k_prefix", "v_prefix", "k", "v", "out")],
        ("lse_strides", ctypes.c_int64 * 2),
        *[(name, ctypes.c_int32) for name in ("B", "Hq", "Hkv", "Nq", "P", "S", "d", "fp8", "causal", "lse_natural")],
        ("softmax_scale", ctypes.c_float),
    ]


def _view(x):
    """``x`` where the kernels can read it: as ``_kernel_view``, with strides of its own along every dimension."""
    x = _kernel_view(x)
    return x if all(st > 0 for st in x.stride()[:3]) else packed_copy(x)


def attn_fwd_shared_prefix(
    q, k_prefix, v_prefix, k, v, q_descale=None, k_descale=None, v_descale=None, k_prefix_descale=None,
    v_prefix_descale=None, causal=False, softmax_scale=None, out=None, return_lse=True, seqused_k=None, lse_natural=False,
):
    """Attend every sequence of a batch to a shared prefix and to its own keys.

    The result is that of ``attn_fwd`` with ``k = cat(k_prefix, own keys)`` for each sequence, but the prefix is read once
    for all sequences: the query rows of the batch go over it together.  For decoding, where a batch continues one long
    prompt; there is no backward.  With many queries a sequence (prompts behind a shared one: from about 64 in FP8 and 128 in
    bf16) and for a few short sequences, ``attn_fwd`` is faster if every sequence has the prefix in front of its own keys.
    FP8 calls take up to twice as long where logits spread widely (by 3 nats and more).

    Args:
        q: ``[B, Hq, Nq, d]`` ``torch.float8_e4m3fn`` or bf16, ``d`` 64 or 128. Strides as for ``attn_fwd``.
        k_prefix: ``[1, Hkv, P, d]``, same dtype. ``Hq`` must be a multiple of ``Hkv``. ``P`` may be 0.
        v_prefix: Same shape and dtype as ``k_prefix``.
        k: ``[B, Hkv, S, d]``, the sequences' own keys. ``S`` may be 0.
        v: Same shape and dtype as ``k``.
        q_descale: ``[B, Hkv]`` float32 dequantization scale, or ``None`` for 1. Descales are positive.
        k_descale: Same as ``q_descale``, for ``k``.
        v_descale: Same as ``q_descale``, for ``v``.
        k_prefix_descale: ``[1, Hkv]``, for ``k_prefix``.
        v_prefix_descale: ``[1, Hkv]``, for ``v_prefix``.
        causal: Whether query ``i`` sees only the first ``P + n - Nq + i + 1`` keys of the prefix and the ``n`` own keys of
            its sequence (the bottom-right aligned mask of ``attn_fwd``).
        softmax_scale: Scale on the logits, positive. Defaults to ``1 / sqrt(d)``.
        out: Output buffer, ``[B, Hq, Nq, d]`` bf16 with last stride 1, such as ``q`` itself; it must not share a byte with
            anything else. ``None`` allocates one with the memory layout of ``q``.
        return_lse: Whether to compute ``lse``.
        seqused_k: ``[B]`` int32, how many of its ``S`` own keys each sequence attends to; ``None`` for all. It is read on
            the device (a captured graph sees later values). What ``k`` and ``v`` hold behind them is never used.
            What a query sees there must be finite, also for the other queries that the causal mask hides it from.
        lse_natural: Whether ``lse`` is the natural-log log-sum-exp instead of base 2.

    Returns:
        ``(out, lse)``: ``out`` ``[B, Hq, Nq, d]`` bf16, ``lse`` the ``[B, Hq, Nq]`` base-2 log-sum-exp of the scaled logits,
        or ``None`` without ``return_lse``. Rows with no visible key get 0 and ``+inf``.

    Raises:
        ValueError: If a dtype, shape, device or option does not fit, or ``out`` overlaps an input without being ``q``.
        NotImplementedError: If the GPU does not support the dtype of ``q``.
    """
    done = _lib.host().attn_fwd_shared_prefix(q, k_prefix, v_prefix, k, v, q_descale, k_descale, v_descale, k_prefix_descale,
                                              v_prefix_descale, causal, softmax_scale, out, return_lse, seqused_k, lse_natural)
    if done is not None:
        return done
    _check_qkv(q, k_prefix, v_prefix)
    _check_qkv(q, k, v)
    fp8 = q.dtype != torch.bfloat16
    require("attn_fwd_shared_prefix", q)
    names = ("q", "k_prefix", "v_prefix", "k", "v")
    tensors = (q, k_prefix, v_prefix, k, v)
    if any(x.dim() != 4 for x in tensors) or q.numel() == 0:
        raise ValueError("need q [B, Hq, Nq, d], k_prefix, v_prefix [1, Hkv, P, d] and k, v [B, Hkv, S, d]")
    if any(not x.is_cuda or x.device != q.device for x in tensors):
        raise ValueError("q, k_prefix, v_prefix, k and v must be on one CUDA device")
    B, Hq, Nq, d = q.shape
    Hkv, P, S = k.shape[1], k_prefix.shape[2], k.shape[2]
    if (d not in (64, 128) or Hkv < 1 or Hq % Hkv or k_prefix.shape != (1, Hkv, P, d) or v_prefix.shape != k_prefix.shape
            or k.shape != (B, Hkv, S, d) or v.shape != k.shape):
        raise ValueError(
            "need q [B, Hq, Nq, d], k_prefix, v_prefix [1, Hkv, P, d] and k, v [B, Hkv, S, d] with d 64 or 128 and Hq a "
            f"multiple of Hkv, got {[tuple(x.shape) for x in tensors]}"
        )
    descales = {"q_descale": (q_descale, B), "k_descale": (k_descale, B), "v_descale": (v_descale, B),
                "k_prefix_descale": (k_prefix_descale, 1), "v_prefix_descale": (v_prefix_descale, 1)}
    if not fp8 and any(x is not None for x, _ in descales.values()):
        raise ValueError("descales apply to float8_e4m3fn inputs only")
    dev = q.device
    for name, (x, rows) in descales.items():
        check_descale(x, rows, Hkv, name)
        if x is not None and x.device != dev:
            raise ValueError(f"{name} must be on the device of q")
    if softmax_scale is None:
        softmax_scale = 1.0 / math.sqrt(d)
    if not softmax_scale > 0:
        raise ValueError("softmax_scale must be positive")
    if seqused_k is not None and (
        seqused_k.shape != (B,) or seqused_k.dtype != torch.int32 or seqused_k.device != dev
    ):
        raise ValueError("seqused_k must be an int32 CUDA tensor of shape [B]")
    if out is None:
        out = torch.empty_like(q, dtype=torch.bfloat16)
    elif out.shape != q.shape or out.dtype != torch.bfloat16 or out.device != dev or out.stride(3) != 1 or not apart(out):
        raise ValueError("out must be a bf16 tensor shaped like q, with last stride 1, whose elements do not share memory")
    else:
        for name, x in zip(names, tensors):
            same = x is tensors[0] and out.data_ptr() == x.data_ptr() and out.stride() == x.stride() and not fp8
            if not same and overlap(out, x):
                raise ValueError(f"out must not overlap {name}" + (" without being it" if name == "q" else ""))
    args = _PrefixArgs()
    views = [_view(x) for x in tensors]
    direct = out.data_ptr() % 8 == 0 and all(st > 0 and st % 4 == 0 for st in out.stride()[:3])
    out_k = out if direct else torch.empty(out.shape, dtype=out.dtype, device=dev)
    for name, x in (*zip(names, views), ("out", out_k)):
        setattr(args, name, x.data_ptr() if x.numel() else None)
        setattr(args, name + "_strides", (ctypes.c_int64 * 3)(*x.stride()[:3]))
    keep = [*views, out_k]
    if fp8:
        for name, (x, rows) in descales.items():
            if x is None:
                x = cached_tensor(("ones", dev, rows, Hkv), lambda: torch.ones(rows, Hkv, dtype=torch.float32, device=dev))
            x = x.float().contiguous()
            setattr(args, name, x.data_ptr())
            keep.append(x)
    seq = None if seqused_k is None else seqused_k.contiguous()
    args.seqused_k = None if seq is None else seq.data_ptr()
    lse = torch.empty(B, Hq, Nq, dtype=torch.float32, device=dev) if return_lse else None
    if return_lse:
        args.lse = lse.data_ptr()
        args.lse_strides = (ctypes.c_int64 * 2)(*lse.stride()[:2])
    args.B, args.Hq, args.Hkv, args.Nq, args.P, args.S, args.d = B, Hq, Hkv, Nq, P, S, d
    args.fp8, args.causal, args.lse_natural = int(fp8), int(bool(causal)), int(bool(lse_natural))
    args.softmax_scale = float(softmax_scale)
    lib = _lib.lib()
    with torch.cuda.device(dev):
        args.workspace_bytes = lib.wk_attn_fwd_shared_prefix_workspace_bytes(B, Hq, Hkv, Nq, P, S, d)
    if args.workspace_bytes == 0:
        raise ValueError("the problem has more than 2^30 query rows, 2^30 keys of a sequence or 2^27 tiles of keys")
    workspace = torch.empty(args.workspace_bytes, dtype=torch.uint8, device=dev)
    args.workspace = workspace.data_ptr()
    entry = _lib.address(lib.wk_attn_fwd_shared_prefix)
    _lib.check(_lib.host().launch(entry, ctypes.addressof(args), dev.index), "attn_fwd_shared_prefix")
    if not direct:
        out.copy_(out_k)
    return out, lse
