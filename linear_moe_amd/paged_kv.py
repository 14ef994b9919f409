"""A paged cache of keys and values on MI355X, and the attention of one new token over it: what the softmax layers of a hybrid
model need while it generates, next to the ``fused_recurrent_*`` ops of its linear layers (the reference's generation keeps
dense caches, ``linear_moe/generation``).

    o = softmax_attn(q, k, v, cu_seqlens=cu, head_first=False)                       # the prompts
    paged_kv_append(k_pages, v_pages, k, v, page_table, zeros, cu_seqlens=cu, head_first=False)
    ...
    o = paged_attn_decode(q, k_pages, v_pages, page_table, lens, k=k, v=v)           # one token of each, written and attended to
    lens += 1

``k_pages`` ``[P, S, HKV, K]`` and ``v_pages`` ``[P, S, HKV, V]``: P pages of S tokens, in any strides that keep 16-byte rows (a
view of ``[P, HKV, S, D]`` is as good).  Position j of sequence n lies in slot ``j % S`` of page ``page_table[n, j // S]``;
``page_table`` ``[N, M]`` and ``lens`` ``[N]`` (tokens in the cache) are int32 on the device and are never read by the host, so a
step captures into a HIP graph and a replay follows what they hold then.  A page number outside 0 .. P - 1 names no page: its
positions take no part and are not written.
"""
from __future__ import annotations

import ctypes as C
from typing import Optional

import torch

from . import _lib
from ._host import _DT, _desc, has_tangent, native_call, ptr, stream_ptr
from .softmax_attn import MAX_DIM, cap_of, has_rows16, ints_of, on_current_device, rows16, slopes_of, to_int32


def _pages(k_pages, v_pages, page_table, lens, name):
    for x, n in ((k_pages, "k_pages"), (v_pages, "v_pages")):
        if x.dim() != 4:
            raise ValueError(f"{name}: {n} must be [P, S, HKV, D], got {tuple(x.shape)}")
    on_current_device(k_pages.device, name)
    dev, dt = k_pages.device, k_pages.dtype
    if dt not in _DT or v_pages.dtype != dt:
        raise ValueError(f"{name}: the pages must share dtype bfloat16 or float32, got {dt}, {v_pages.dtype}")
    if k_pages.shape[:3] != v_pages.shape[:3] or v_pages.device != dev:
        raise ValueError(f"{name}: k_pages {tuple(k_pages.shape)} and v_pages {tuple(v_pages.shape)} must agree in pages, tokens and heads")
    P, S, HKV, K = k_pages.shape
    V = v_pages.shape[3]
    step = 16 // k_pages.element_size()
    if not (0 < K <= MAX_DIM and 0 < V <= MAX_DIM) or K % step or V % step:
        raise ValueError(f"{name}: head dimensions K={K}, V={V} unsupported (multiples of {step} up to {MAX_DIM})")
    if S < 1 or HKV < 1:
        raise ValueError(f"{name}: pages of {S} tokens and {HKV} heads")
    if not (has_rows16(k_pages) and has_rows16(v_pages)):
        raise ValueError(f"{name}: the pages must keep 16-byte aligned rows (they are used in place)")
    if page_table.dim() != 2 or page_table.is_floating_point() or page_table.is_complex() or page_table.dtype == torch.bool or page_table.device != dev:
        raise ValueError(f"{name}: page_table must be [N, M] whole numbers on {dev}, got {tuple(page_table.shape)} of {page_table.dtype} on "
                         f"{page_table.device}")
    if page_table.dtype != torch.int32 or (page_table.shape[1] > 1 and page_table.stride(1) != 1):
        page_table = to_int32(page_table).contiguous()
    N, M = page_table.shape
    lens = ints_of(lens, N, dev, f"{name}: lens")
    a = _lib.PagedArgs()
    a.dtype, a.N, a.HKV, a.K, a.V, a.P, a.S, a.M = _DT[dt], N, HKV, K, V, P, S, M
    a.table_stride, a.table, a.lens = page_table.stride(0), page_table.data_ptr(), lens.data_ptr()
    a.kp, a.vp = (_lib.Tensor4(x.data_ptr(), x.stride(0), x.stride(1), x.stride(2)) for x in (k_pages, v_pages))
    return a, (page_table, lens)


def _tokens(x, B, T, H, D, head_first, like, name):
    """New tokens as the kernels read them."""
    want = (B, H, T, D) if head_first else (B, T, H, D)
    if tuple(x.shape) != want:
        raise ValueError(f"{name} must have shape {want}, got {tuple(x.shape)}")
    if x.dtype != like.dtype or x.device != like.device:
        raise ValueError(f"{name} must be {like.dtype} on {like.device} like the pages, got {x.dtype} on {x.device}")
    return rows16(x.detach())


def _no_grad(name, *xs):
    if torch.is_grad_enabled() and any(x is not None and x.requires_grad for x in xs):
        raise RuntimeError(f"{name} is for generation and has no backward: call it under torch.no_grad(), or train with softmax_attn")
    if any(x is not None and has_tangent(x) for x in xs):
        raise RuntimeError(f"{name} is for generation and has no forward-mode derivative")
    if torch._C._get_tracing_state() is not None:
        raise RuntimeError(f"{name} cannot be recorded in a trace, which would hold its allocations alone")


def _written(*pages):
    """Autograd's count of writes (a backward that saved the pages notices them)."""
    for x in pages:
        if not x.is_inference():
            torch.autograd.graph.increment_version(x)


def paged_attn_decode(
    q: torch.Tensor,
    k_pages: torch.Tensor,
    v_pages: torch.Tensor,
    page_table: torch.Tensor,
    lens: torch.Tensor,
    k: Optional[torch.Tensor] = None,
    v: Optional[torch.Tensor] = None,
    scale: Optional[float] = None,
    softcap: Optional[float] = None,
    slopes: Optional[torch.Tensor] = None,
    head_first: bool = True,
) -> torch.Tensor:
    """Attention of one new token per sequence: q ``[N,HQ,1,K]`` (``[N,1,HQ,K]`` with ``head_first=False``) over the ``lens[n]`` tokens
    of the cache and, where its own k and v are given (shaped like q with HKV heads), itself; these are written into the cache at position
    ``lens[n]`` by the same launch (``lens`` itself is the caller's to advance).  Returns o ``[N,HQ,1,V]`` / ``[N,1,HQ,V]``.

    scale, softcap, slopes as in ``softmax_attn``; distances count to the new token (the last in the cache where k is not given).  A
    sequence with nothing to attend to gives zeros.  A position beyond the table is attended to but not kept."""
    name = "paged_attn_decode"
    _no_grad(name, q, k, v, k_pages, v_pages, slopes)
    r = native_call("paged_decode", name, k_pages, v_pages, page_table, lens, q, k, v, scale, softcap, slopes, head_first)
    if r is not None:
        return r[0]
    if (k is None) != (v is None):
        raise ValueError(f"{name}: k and v go together")
    a, held = _pages(k_pages, v_pages, page_table, lens, name)
    if q.dim() != 4:
        raise ValueError(f"{name}: q must be 4-dimensional")
    HQ = q.shape[1 if head_first else 2]
    if HQ < 1 or HQ % a.HKV:
        raise ValueError(f"{name}: {HQ} query heads are no multiple of {a.HKV} key heads")
    q = _tokens(q, a.N, 1, HQ, a.K, head_first, k_pages, f"{name}: q")
    a.HQ, a.q = HQ, _desc(q, head_first)
    if k is not None:
        k, v = (_tokens(x, a.N, 1, a.HKV, d, head_first, k_pages, f"{name}: {s}") for x, d, s in ((k, a.K, "k"), (v, a.V, "v")))
        a.kn, a.vn = _desc(k, head_first), _desc(v, head_first)
    a.scale, a.softcap = float(a.K ** -0.5 if scale is None else scale), cap_of(softcap, name)
    slopes = slopes_of(slopes, HQ, q.device, name)
    a.slopes = ptr(slopes)
    o = torch.empty((*q.shape[:3], a.V), dtype=q.dtype, device=q.device)
    a.o = _desc(o, head_first)
    if a.N == 0:
        return o
    lib = _lib.load()
    floats = lib.lmoe_paged_attn_floats(C.byref(a))
    _lib.check(min(floats, 0), name)
    ws = torch.empty(floats, dtype=torch.float32, device=q.device) if floats else None
    a.ws = ptr(ws)
    _lib.check(lib.lmoe_paged_attn_decode(C.byref(a), stream_ptr()), name)
    if k is not None:
        _written(k_pages, v_pages)
    return o


def paged_kv_append(
    k_pages: torch.Tensor,
    v_pages: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    page_table: torch.Tensor,
    lens: torch.Tensor,
    cu_seqlens: Optional[torch.Tensor] = None,
    head_first: bool = True,
) -> None:
    """Writes k ``[N,HKV,T,K]`` and v ``[N,HKV,T,V]`` (``[N,T,H,*]`` with ``head_first=False``; packed ``[1,T,H,*]`` with ``cu_seqlens``) into
    the cache: token t of sequence n goes to position ``lens[n] + t``.  ``lens`` itself is the caller's to advance.  Tokens behind the
    last packed sequence, and positions that have no page, are left out."""
    name = "paged_kv_append"
    _no_grad(name, k, v, k_pages, v_pages)
    if native_call("paged_append", name, k_pages, v_pages, page_table, lens, k, v, cu_seqlens, head_first) is not None:
        return
    a, held = _pages(k_pages, v_pages, page_table, lens, name)
    if k.dim() != 4 or v.dim() != 4:
        raise ValueError(f"{name}: k and v must be 4-dimensional")
    cu = None
    if cu_seqlens is not None:
        if head_first:
            raise ValueError("cu_seqlens requires head_first=False ([1, T, H, D] packed input)")
        if k.shape[0] != 1:
            raise ValueError(f"cu_seqlens requires batch size 1 (packed input), got B={k.shape[0]}")
        if cu_seqlens.dim() != 1 or cu_seqlens.numel() != a.N + 1:
            raise ValueError(f"{name}: cu_seqlens must hold {a.N + 1} offsets for the {a.N} rows of page_table, got {tuple(cu_seqlens.shape)}")
        if not cu_seqlens.is_cuda:
            offs = cu_seqlens.detach().to(torch.int64)
            if int(offs[0]) != 0 or int(offs[-1]) != k.shape[1] or bool((offs[1:] < offs[:-1]).any()):
                raise ValueError("cu_seqlens must start at 0, be non-decreasing and end at T")
        cu = cu_seqlens.detach().to(device=k_pages.device, dtype=torch.int32).contiguous()
        a.cu_seqlens = cu.data_ptr()
    B, T = (1 if cu is not None else a.N), k.shape[2 if head_first else 1]
    k, v = (_tokens(x, B, T, a.HKV, d, head_first, k_pages, f"{name}: {s}") for x, d, s in ((k, a.K, "k"), (v, a.V, "v")))
    a.B, a.T, a.kn, a.vn = B, T, _desc(k, head_first), _desc(v, head_first)
    if k.numel() and a.N:
        _lib.check(_lib.load().lmoe_paged_kv_append(C.byref(a), stream_ptr()), name)
        _written(k_pages, v_pages)
