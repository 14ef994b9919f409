"""Softmax attention on MI355X: the layers that a hybrid model keeps between its linear ones.

The reference's hybrid blocks mix linear ('L') and softmax ('N') layers
(``linear_moe/model/qwen2/hybrid/hybrid_transformer_block.py:149-165``); the core of the latter is
``linear_moe/sequence_modeling/attention/dot_product_attention.py:139-183``, which forms the whole matrix of scores in
memory.  Here one kernel forms the output with a running maximum and sum, and two form the gradients from the sums it kept;
nothing of the size of the scores reaches memory.  Layouts, ``scale``, ``cu_seqlens`` and ``head_first`` are those of the
chunk ops.
"""
from __future__ import annotations

import ctypes as C
from typing import Optional

import torch
from torch.autograd.function import once_differentiable

from . import _lib
from ._host import _DT, _desc, has_tangent, native_call, no_node, no_transform, ptr, seq_plan, stream_ptr

MAX_DIM = 128      # columns of a head


def slopes_of(slopes, H: int, device, name: str):
    if slopes is None:
        return None
    if slopes.requires_grad and torch.is_grad_enabled():
        raise ValueError(f"{name}: slopes are constants of the model, there is no gradient for them")
    if has_tangent(slopes):
        raise RuntimeError(f"{name}: slopes are constants of the model, there is no forward-mode derivative for them")
    if slopes.numel() != H or slopes.device != device:
        raise ValueError(f"{name}: slopes must be {H} numbers on {device}, got {tuple(slopes.shape)} on {slopes.device}")
    return slopes.detach().reshape(H).to(torch.float32).contiguous()


def cap_of(softcap, name: str) -> float:
    cap = 0.0 if softcap is None else float(softcap)
    if not 0.0 <= cap < 3e38:
        raise ValueError(f"{name}: softcap must be positive, or 0 / None for none, got {softcap}")
    return max(cap, 2.0 ** -126) if cap else 0.0         # (the kernels hold it in 32 bits, where 0 is none)


def to_int32(x: torch.Tensor) -> torch.Tensor:
    """Whole numbers in 32 bits; what those do not hold becomes the nearest they do (out of any range all the same)."""
    wide = x.dtype in (torch.int64, torch.uint32, torch.uint64)
    return (x.to(torch.int64).clamp(-2 ** 31, 2 ** 31 - 1) if wide else x).to(torch.int32)


def ints_of(x: torch.Tensor, n: int, device, name: str) -> torch.Tensor:
    """One whole number per sequence, as the kernels read them."""
    if x.dim() != 1 or x.numel() != n or x.is_floating_point() or x.is_complex() or x.dtype == torch.bool:
        raise ValueError(f"{name} must be {n} whole numbers, got {tuple(x.shape)} of {x.dtype}")
    if x.device != device:
        raise ValueError(f"{name} must live on {device}, got {x.device}")
    return to_int32(x.detach()).contiguous()


def on_current_device(device, name: str) -> None:
    if device.type != "cuda":
        raise RuntimeError(f"{name}: linear_moe_amd ops run on the GPU only (HIP kernels; there is no CPU path)")
    if device.index != torch._C._cuda_getDevice():
        raise RuntimeError(f"{name}: the tensors must live on the current device cuda:{torch.cuda.current_device()}, got {device}")


def has_rows16(x: torch.Tensor) -> bool:
    s = x.stride()
    return s[3] == 1 and x.data_ptr() % 16 == 0 and (s[0] | s[1] | s[2]) % (16 // x.element_size()) == 0


def rows16(x: torch.Tensor) -> torch.Tensor:
    """x, or a copy of it, with contiguous rows on 16-byte boundaries."""
    return x if has_rows16(x) else x.clone(memory_format=torch.contiguous_format)


def _check(q, k, v, head_first, cu_seqlens):
    name = "softmax_attn"
    if q.dim() != 4 or k.dim() != 4 or v.dim() != 4:
        raise ValueError(f"{name}: q, k, v must be 4-dimensional")
    if not (q.is_cuda and k.is_cuda and v.is_cuda):
        raise RuntimeError("linear_moe_amd ops run on the GPU only (HIP kernels; there is no CPU path)")
    if q.dtype not in _DT or k.dtype != q.dtype or v.dtype != q.dtype:
        raise ValueError(f"{name}: q, k, v must share dtype bfloat16 or float32, got {q.dtype}, {k.dtype}, {v.dtype}")
    h, t = (1, 2) if head_first else (2, 1)
    B, T, HQ, K = q.shape[0], q.shape[t], q.shape[h], q.shape[3]
    HKV, V = k.shape[h], v.shape[3]
    if (k.shape[0], k.shape[t], k.shape[3]) != (B, T, K) or k.shape[:3] != v.shape[:3]:
        raise ValueError(f"{name}: shape mismatch: q {tuple(q.shape)}, k {tuple(k.shape)}, v {tuple(v.shape)}")
    if HQ < 1 or HKV < 1 or HQ % HKV:
        raise ValueError(f"{name}: {HQ} query heads are no multiple of {HKV} key heads")
    if not (0 < K <= MAX_DIM and 0 < V <= MAX_DIM):
        raise ValueError(f"{name}: head dimensions K={K}, V={V} unsupported (1 to {MAX_DIM})")
    if cu_seqlens is not None:
        if head_first:
            raise ValueError("cu_seqlens requires head_first=False ([1, T, H, D] packed input)")
        if B != 1:
            raise ValueError(f"cu_seqlens requires batch size 1 (packed input), got B={B}")
    return B, T, HQ, HKV, K, V


def _args(q, k, v, o, lse, low, dims, head_first, scale, causal, softcap, slopes, prefix, plan):
    B, T, HQ, HKV, K, V = dims
    a = _lib.AttnArgs()
    a.dtype, a.causal = _DT[q.dtype], int(causal)
    a.B, a.T, a.HQ, a.HKV, a.K, a.V, a.N, a.NT = B, T, HQ, HKV, K, V, plan.N, plan.NT
    a.scale, a.softcap = scale, softcap
    if plan.cu is not None:
        a.cu_seqlens, a.chunk_map, a.nt_dev, a.seq_order = (plan.cu.data_ptr(), plan.chunk_map.data_ptr(), ptr(plan.nt_dev),
                                                            ptr(plan.seq_order))
    a.slopes, a.prefix_lens = ptr(slopes), ptr(prefix)
    a.q, a.k, a.v, a.o = (_desc(x, head_first) for x in (q, k, v, o))
    a.lse, a.o_low = ptr(lse), ptr(low)
    return a


def _forward(q, k, v, dims, head_first, scale, causal, softcap, slopes, prefix, plan, save):
    B, T, HQ, HKV, K, V = dims
    r = native_call("attn_forward", "softmax_attn forward", q, k, v, scale, causal, softcap, slopes, prefix, plan.tables, head_first, save)
    if r is not None:
        return (q, k, v, *r)
    q, k, v = rows16(q.detach()), rows16(k.detach()), rows16(v.detach())
    o = torch.empty((*q.shape[:3], V), dtype=q.dtype, device=q.device)
    lse = torch.empty(B, HQ, T, dtype=torch.float32, device=q.device) if save else None
    low = torch.empty(B, HQ, T * V, dtype=torch.int8, device=q.device) if save and q.dtype == torch.bfloat16 else None
    if B * T:
        a = _args(q, k, v, o, lse, low, dims, head_first, scale, causal, softcap, slopes, prefix, plan)
        _lib.check(_lib.load().lmoe_softmax_attn_fwd(C.byref(a), stream_ptr()), "softmax_attn forward")
    return q, k, v, o, lse, low


def _back(x, shape, dtype, device, name):
    """A tensor that was saved for the backward, as the kernels may read it (a saved-tensor hook hands back what it likes)."""
    if x is None or tuple(x.shape) != tuple(shape) or x.device != device:
        raise RuntimeError(f"{name}, saved for the backward with shape {tuple(shape)} on {device}, came back as "
                           f"{None if x is None else (tuple(x.shape), str(x.device))}")
    return rows16(x.to(dtype)) if x.dim() == 4 else x.to(dtype).contiguous()


class _SoftmaxAttn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, dims, head_first, scale, causal, softcap, slopes, prefix, plan):
        qs, ks, vs, o, lse, low = _forward(q, k, v, dims, head_first, scale, causal, softcap, slopes, prefix, plan, True)
        ctx.save_for_backward(qs, ks, vs, o, lse, low, slopes, prefix)
        ctx.call = dims, head_first, scale, causal, softcap, plan
        ctx.shapes, ctx.dtype, ctx.options = (q.shape, k.shape, v.shape, o.shape), q.dtype, (slopes is not None, prefix is not None)
        return o

    @staticmethod
    @once_differentiable
    def backward(ctx, do):
        dims, head_first, scale, causal, softcap, plan = ctx.call
        B, T, HQ, HKV, K, V = dims
        q, k, v, o, lse, low, slopes, prefix = ctx.saved_tensors
        keys = any(ctx.needs_input_grad[1:3])
        if (q.shape, k.shape, v.shape, o.shape) == ctx.shapes and (slopes is not None, prefix is not None) == ctx.options:
            r = native_call("attn_backward", "softmax_attn backward", q, k, v, scale, causal, softcap, slopes, prefix, plan.tables,
                            head_first, o, lse, low, do, keys)
            if r is not None:
                return (*r, *(None,) * 8)
        dev, dt = do.device, ctx.dtype
        q, k, v, o = (_back(x, s, dt, dev, n) for x, s, n in zip((q, k, v, o), ctx.shapes, "qkvo"))
        do = _back(do, ctx.shapes[3], dt, dev, "the gradient")
        lse = _back(lse, (B, HQ, T), torch.float32, dev, "lse")
        if dt == torch.bfloat16:
            low = _back(low, (B, HQ, T * V), torch.int8, dev, "o_low")
        if ctx.options[0]:
            slopes = _back(slopes, (HQ,), torch.float32, dev, "slopes")
        if ctx.options[1]:
            prefix = _back(prefix, (plan.N,), torch.int32, dev, "prefix_lens")
        dq = torch.empty_like(q)
        dk, dv = (torch.empty_like(k), torch.empty_like(v)) if keys else (None, None)
        if B * T:
            a = _args(q, k, v, o, lse, low, dims, head_first, scale, causal, softcap, slopes, prefix, plan)
            delta = torch.empty(B, HQ, T, dtype=torch.float32, device=dev)
            a.d_o, a.dq, a.dk, a.dv, a.delta = (_desc(do, head_first), _desc(dq, head_first), _desc(dk, head_first),
                                                _desc(dv, head_first), delta.data_ptr())
            lib = _lib.load()
            floats = lib.lmoe_softmax_attn_bwd_floats(C.byref(a))
            _lib.check(min(floats, 0), "softmax_attn backward")
            ws = torch.empty(floats, dtype=torch.float32, device=dev) if floats else None
            a.ws = ptr(ws)
            _lib.check(lib.lmoe_softmax_attn_bwd(C.byref(a), stream_ptr()), "softmax_attn backward")
        return (dq, dk, dv) + (None,) * 8


def softmax_attn(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    scale: Optional[float] = None,
    causal: bool = True,
    softcap: Optional[float] = None,
    slopes: Optional[torch.Tensor] = None,
    prefix_lens: Optional[torch.Tensor] = None,
    cu_seqlens: Optional[torch.Tensor] = None,
    head_first: bool = True,
) -> torch.Tensor:
    """``o_i = sum_j softmax_j(s_ij) v_j``, ``x_ij = scale q_i . k_j``, ``s_ij = softcap tanh(x_ij / softcap) - slope_h |i - j|``.

    q ``[B,HQ,T,K]``, k ``[B,HKV,T,K]``, v ``[B,HKV,T,V]`` (``[B,T,H,*]`` with ``head_first=False``), bfloat16 or float32, any
    strides; HQ a multiple of HKV: query head h reads key head ``h // (HQ // HKV)``.  K, V up to 128 (others than multiples of
    16 bytes are padded).  Returns o, laid out like q with V columns.

    scale: ``None`` is ``K ** -0.5``.  softcap, slopes (``[HQ]``, not trained): as in the formula, left out where ``None`` (or 0).  A cap may be
    any number below 3e38 (less than 2^-126 counts as that, more than 2^100 as that).  Scores are held in float32: up to 2^28 in size.
    causal: row i sees j <= i; prefix_lens (``[N]`` whole numbers on the device, clamped to the sequence's length): and every
    j < its sequence's prefix.  ``causal=False``: all.
    The backward takes a workspace of fp32 sums where several work-groups share a tile of keys: 1 GiB at most, none where the tiles fill the card a few times.
    cu_seqlens: packed documents as in the chunk ops; rows of one never see another's (nor what it holds: a NaN stays in its
    document).  Rows behind the last document are zero in o and in the gradients.
    Without atomics: the gradients of a key head are summed over its query heads in a fixed order.  A NaN or infinity in the k or v of a
    token stays out of the outputs of rows that do not see it; out of their gradients it stays in another document only.
    Forward and backward capture into a HIP graph; capture with leaves of which no graph of an eager step lives any more (torch's
    accumulation nodes belong to the stream of their first use)."""
    grad = not no_node(q, k, v)
    node = grad and no_transform()                   # (a node of the graph, in native code)
    if cu_seqlens is None and (node or not grad):    # (what the native path takes as it is, it also checks)
        call = q, k, v, scale, causal, softcap, slopes, prefix_lens, None, head_first
        r = native_call("attn_node", "softmax_attn", *call) if node else native_call("attn_forward", "softmax_attn forward", *call, False)
        if r is not None:
            return r[0]
    dims = _check(q, k, v, head_first, cu_seqlens)
    B, T, HQ, HKV, K, V = dims
    on_current_device(q.device, "softmax_attn")
    if not (q.device == k.device == v.device):
        raise RuntimeError(f"softmax_attn: q, k, v must live on one device, got {q.device}, {k.device}, {v.device}")
    sc = float(K ** -0.5 if scale is None else scale)
    cap = cap_of(softcap, "softmax_attn")
    slopes = slopes_of(slopes, HQ, q.device, "softmax_attn")
    plan = seq_plan(B, T, cu_seqlens, q.device)
    if prefix_lens is not None:
        if not causal:
            raise ValueError("softmax_attn: prefix_lens belongs to a causal call")
        prefix_lens = ints_of(prefix_lens, plan.N, q.device, "softmax_attn: prefix_lens")
    step = 16 // q.element_size()
    if K % step or V % step:                       # (zero columns change neither the scores nor the other columns)
        pad = torch.nn.functional.pad
        q, k, v = pad(q, (0, -K % step)), pad(k, (0, -K % step)), pad(v, (0, -V % step))
        dims = B, T, HQ, HKV, q.shape[3], v.shape[3]
    rest = dims, head_first, sc, bool(causal), cap, slopes, prefix_lens, plan
    if grad:
        r = native_call("attn_node", "softmax_attn", q, k, v, *rest[2:7], plan.tables, head_first) if node else None
        o = _SoftmaxAttn.apply(q, k, v, *rest) if r is None else r[0]
    else:
        o = _forward(q, k, v, *rest, save=False)[3]
    return o if o.shape[3] == V else o[..., :V]
