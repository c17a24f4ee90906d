"""Paged K/V cache and the operators on it, for streams longer than the 32-frame window, for
sessions that branch, and for any head layout.

Functions over plain tensors (each one call into ``liboasis_b200.so`` on the current stream):

* :func:`qk_norm_rope`, :func:`qk_norm_rope_append` - RMS norm of every query and key head and
  the rotation over several position axes (time, height, width) in one pass; the second also
  writes keys and values into cache pages.
* :func:`attn_window` - attention of packed queries over cache pages with a sliding window of
  frames and a few sink frames that stay visible (``frame_tokens=1``: the token-wise form).
* :func:`copy_pages` - page copies for every layer, keys and values, in one launch.

:class:`PagedKVCacheB200` keeps the pages and their book: sessions own lists of pages, forks share
pages until one of them writes (copy on write), eviction frees what the window has left behind,
compaction moves the used pages to the front.  :class:`PagedBatchB200` is one step's plan.

The operators compute results only: tensors that require gradients, or carry forward-mode tangents, are refused.
The reference keeps whole tensors per session and concatenates each new frame
(``kv_cache/manager.py:246-306``, ``:416-480``) and branches by copying all of it
(``snapshot``/``restore``, ``:555-588``).
"""

from __future__ import annotations

import contextlib
import ctypes
import operator
import struct
import weakref
from typing import Dict, List, Optional, Sequence, Tuple, Union

import numpy as np
import torch
from torch.autograd import forward_ad

from . import _native as N
from .kv_cache import HEAD_DIM, HEADS

_DTYPES = {torch.bfloat16: N.DT_BF16, torch.float16: N.DT_FP16, torch.float32: N.DT_FP32}
_BIG = 0x3fffffff
_CONTIGUOUS = torch.contiguous_format

# the argument structs of include/oasis_b200.h, in native layout
_ROPE = struct.Struct("@5P10q7if3PiP5iPP")
_ATTN = struct.Struct("@3P4q2P5iPi2P8if")
_entries: dict = {}


def _entry(name: str):
    fn = _entries.get(name)
    if fn is None:
        fn = _entries[name] = N.packed_call(name)
    return fn


_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (
    lambda index: torch.cuda.current_stream(index).cuda_stream)
_current_device = getattr(torch._C, "_cuda_getDevice", None) or torch.cuda.current_device


def _dual_level() -> bool:
    """Whether tensors may carry forward-mode tangents."""
    return getattr(forward_ad, "_current_level", 0) >= 0


# Every function first looks at its arguments with one cheap condition; where that does not
# hold, the checks below find out why (or that all is well after all).


def _elsewhere(device: torch.device, stream) -> Optional[object]:
    """The context a call has to be made in: another stream than the current one, or another
    device; None where the current ones are meant."""
    if device.type != "cuda":
        return None
    if stream is not None:
        if stream.device != device:
            raise ValueError(f"the stream is on {stream.device}, the tensors on {device}")
        return torch.cuda.stream(stream)
    if device.index != torch.cuda.current_device():
        return torch.cuda.device(device)
    return None


def _cuda(name: str, t: torch.Tensor, device: Optional[torch.device] = None) -> None:
    if not t.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor")
    if device is not None and t.device != device:
        raise ValueError(f"{name} is on {t.device}, the queries on {device}")


def _heads3(name: str, t: torch.Tensor) -> None:
    if t.dim() != 3 or (t.shape[2] > 1 and t.stride(2) != 1):
        raise ValueError(f"{name} must be [tokens][heads][head_dim] with contiguous head_dim")


def _no_grad(*tensors) -> None:
    grad, dual = torch.is_grad_enabled(), _dual_level()
    for t in tensors:
        if t is not None and (grad and t.requires_grad or dual and forward_ad.unpack_dual(t).tangent is not None):
            raise ValueError("no gradient is computed here: detach the inputs or use torch.no_grad()")


def _index32(name: str, t: torch.Tensor, shape, device) -> None:
    if t.dtype != torch.int32 or tuple(t.shape) != shape or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous int32 tensor of shape {shape}")
    _cuda(name, t, device)


def _pages(k: torch.Tensor, v: torch.Tensor, dims: Sequence[int]) -> None:
    if k.dim() not in dims or k.shape != v.shape or k.dtype != v.dtype:
        raise ValueError("k_pages and v_pages must be alike, [(layers)][pages][kv_heads][page_tokens][head_dim]")
    if k.dtype not in (torch.bfloat16, torch.float16):
        raise ValueError("cache pages are bf16 or fp16")
    if not (k.is_contiguous() and v.is_contiguous()):
        raise ValueError("cache pages must be contiguous")


def rope_axis_freqs(axes: Sequence[int], theta: Union[float, Sequence[float]] = 10000.0,
                    device="cuda") -> torch.Tensor:
    """fp64 angular frequencies of every rotated pair: axis ``a`` of ``d = axes[a]`` dims has
    the ``d / 2`` frequencies ``theta ** (-2 i / d)`` (``theta`` may be one per axis)."""
    thetas = [float(theta)] * len(axes) if isinstance(theta, (int, float)) else [float(t) for t in theta]
    if len(thetas) != len(axes):
        raise ValueError("one theta per axis")
    if not axes or any(d <= 0 or d % 2 for d in axes) or any(not t > 0 for t in thetas):
        raise ValueError("axes are even numbers of dims, theta is positive")
    parts = [t ** (-2.0 * np.arange(d // 2) / d) for d, t in zip(axes, thetas)]
    return torch.from_numpy(np.concatenate(parts)).to(device)


def _rope_checks(q, k, v, positions, freqs, q_weight, k_weight, axes, norm, k_pages, v_pages, slots) -> None:
    _heads3("q", q)
    _heads3("k", k)
    _cuda("q", q)
    dev = q.device
    _cuda("k", k, dev)
    tokens, _, d = q.shape
    if k.shape[0] != tokens or k.shape[2] != d or k.dtype != q.dtype:
        raise ValueError("q and k must agree in tokens, head_dim and type")
    if q.dtype not in _DTYPES:
        raise ValueError("q and k must be bf16, fp16 or fp32")
    n_axes = len(axes)
    if not 1 <= n_axes <= N.MAX_AXES:
        raise ValueError("1 to 4 position axes")
    shape = tuple(positions.shape)
    if (positions.dtype not in (torch.int32, torch.int64) or not positions.is_contiguous()
            or not (shape == (tokens, n_axes) or (n_axes == 1 and shape == (tokens,)))):
        raise ValueError(f"positions must be contiguous int32 or int64 [{tokens}][{n_axes}]")
    _cuda("positions", positions, dev)
    if freqs.dtype != torch.float64 or freqs.dim() != 1 or 2 * freqs.shape[0] != sum(axes) or not freqs.is_contiguous():
        raise ValueError("freqs must be a contiguous fp64 tensor of sum(axes) / 2 frequencies")
    _cuda("freqs", freqs, dev)
    for name, w in (("q_weight", q_weight), ("k_weight", k_weight)):
        if w is not None:
            if not norm:
                raise ValueError(f"{name} without the norm")
            if w.dtype != torch.float32 or tuple(w.shape) != (d,) or not w.is_contiguous():
                raise ValueError(f"{name} must be a contiguous fp32 tensor [{d}]")
            _cuda(name, w, dev)
    if v is not None:
        _heads3("v", v)
        if v.shape != k.shape or v.dtype != k.dtype:
            raise ValueError("v must have k's shape and type")
        _cuda("v", v, dev)
        _pages(k_pages, v_pages, (4,))
        _cuda("k_pages", k_pages, dev)
        _cuda("v_pages", v_pages, dev)
        if k_pages.shape[1] != k.shape[1] or k_pages.shape[3] != d or k_pages.dtype != k.dtype:
            raise ValueError("the pages do not fit the keys (kv_heads, head_dim, type)")
        _index32("slots", slots, (tokens,), dev)
    _no_grad(q, k, v, freqs, q_weight, k_weight, k_pages, v_pages)


def _starts(t: torch.Tensor) -> np.ndarray:
    """Byte addresses of a view's [tokens][heads] runs of head_dim elements."""
    (n, h, _), (ts, hs, _), e = t.shape, t.stride(), t.element_size()
    return t.data_ptr() + e * (ts * np.arange(n)[:, None] + hs * np.arange(h)).ravel()


def _extent(shape, strides, size: int) -> int:
    """Bytes from a tensor's first element to behind its last."""
    n = 1
    for m, st in zip(shape, strides):
        if m == 0:
            return 0
        n += st * (m - 1)
    return n * size


def _overlap(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether two [tokens][heads][head_dim] views (head_dim contiguous), or such a view and a contiguous tensor, have
    memory in common.  Exact: columns of one projection interleave and have none."""
    x, y, e = a.data_ptr(), b.data_ptr(), a.element_size()
    sa, sb, ta, tb = a.shape, b.shape, a.stride(), b.stride()
    if x >= y + _extent(sb, tb, b.element_size()) or y >= x + _extent(sa, ta, e):
        return False
    step = ta[0] * e
    same_step = step > 0 and len(sb) == 3 and step == tb[0] * e
    if same_step:  # the usual case: each token's heads lie in a part of the step of their own
        at = (y - x) % step
        if at >= _extent(sa[1:], ta[1:], e) and at + _extent(sb[1:], tb[1:], e) <= step:
            return False
    if a.is_contiguous() and b.is_contiguous():
        return True
    a, b = (t if t.dim() == 3 else t.view(1, 1, -1) for t in (a, b))
    da, db = (t.shape[2] * t.element_size() for t in (a, b))
    if same_step:
        # runs of token i and head j of a, token k and head l of b: only i - k counts; for each of the heads the
        # nearest multiples of the step that are within the tokens
        gap = _starts(b[:1])[None] - _starts(a[:1])[:, None]
        lo, hi = 1 - b.shape[0], a.shape[0] - 1
        near = gap // step
        return any(bool(((off > -db) & (off < da)).any())
                   for u in (near, near + 1) for off in (gap - step * np.clip(u, lo, hi),))
    first, second = _starts(a), np.sort(_starts(b))  # any strides
    at = np.searchsorted(second, first)
    before, after = second[np.maximum(at - 1, 0)], second[np.minimum(at, len(second) - 1)]
    return bool((((before <= first) & (before + db > first)) | ((after >= first) & (after < first + da))).any())


def _folds(t: torch.Tensor) -> bool:
    """Whether a view's rows lie over one another."""
    (n, h, d), (ts, hs, _) = t.shape, t.stride()
    for (n1, s1), (n2, s2) in (((n, ts), (h, hs)), ((h, hs), (n, ts))):
        if (n2 <= 1 or s2 >= d) and (n1 <= 1 or s1 >= (s2 * (n2 - 1) if n2 > 1 else 0) + d):
            return False  # the usual layouts: one dimension's rows lie within a step of the other
    at = np.sort(_starts(t))
    return bool((np.diff(at) < d * t.element_size()).any())


def _out_check(name: str, out: torch.Tensor, like: torch.Tensor, **others: Optional[torch.Tensor]) -> None:
    """An output given: like its input, over it exactly or not at all, and off the other tensors."""
    if out is not like:
        if out.shape != like.shape or out.dtype != like.dtype or out.device != like.device:
            raise ValueError(f"{name} must have its input's shape, type and device")
        _no_grad(out)
        _heads3(name, out)
    shape, strides = out.shape, out.stride()
    if 0 in strides and any(st == 0 and n > 1 for st, n in zip(strides, shape)):
        raise ValueError(f"{name} must not be an expanded tensor: its rows are one memory")
    at = out.data_ptr()
    if out is not like and at == like.data_ptr() and strides != like.stride():
        raise ValueError(f"{name} over its input must have the input's strides")
    if _folds(out):
        raise ValueError(f"{name}'s rows overlap each other")
    end = at + _extent(shape, strides, out.element_size())
    if out is not like and like.data_ptr() != at:
        others["its input, except to lie over it exactly"] = like
    for other, t in others.items():
        if t is not None and t.data_ptr() < end and _overlap(out, t):
            raise ValueError(f"{name} must not overlap {other}")


def _rope(q, k, v, positions, freqs, k_pages, v_pages, slots, axes, interleaved, norm, q_weight, k_weight, eps,
          q_out, k_out):
    dev, dt = q.get_device(), q.dtype
    qh, kh, ph = q.shape, k.shape, positions.shape
    n_axes, pt = len(axes), positions.dtype
    fine = (dev >= 0 and dev == k.get_device() == positions.get_device() == freqs.get_device()
            and len(qh) == len(kh) == 3 and qh[0] == kh[0] and qh[2] == kh[2] and dt == k.dtype and dt in _DTYPES
            and 1 <= n_axes <= 4 and (pt is torch.int32 or pt is torch.int64) and ph == (qh[0], n_axes)
            and freqs.dtype is torch.float64 and freqs.dim() == 1 and 2 * freqs.numel() == sum(axes)
            and positions.is_contiguous() and freqs.is_contiguous()
            and not (q.requires_grad or k.requires_grad or freqs.requires_grad or _dual_level())
            and q_weight is not None and k_weight is not None and norm
            and q_weight.dtype is k_weight.dtype is torch.float32 and q_weight.shape == k_weight.shape == qh[2:]
            and q_weight.get_device() == k_weight.get_device() == dev
            and q_weight.is_contiguous() and k_weight.is_contiguous()
            and not (q_weight.requires_grad or k_weight.requires_grad))
    if fine and v is not None:
        gh = k_pages.shape
        fine = (v.get_device() == k_pages.get_device() == v_pages.get_device() == slots.get_device() == dev
                and v.shape == kh and v.dtype == dt == k_pages.dtype == v_pages.dtype and dt is not torch.float32
                and len(gh) == 4 and gh == v_pages.shape and gh[1] == kh[1] and gh[3] == kh[2]
                and k_pages.is_contiguous() and v_pages.is_contiguous() and slots.dtype is torch.int32
                and slots.shape == qh[:1] and slots.is_contiguous()
                and not (v.requires_grad or k_pages.requires_grad or v_pages.requires_grad))
    if not fine:
        _rope_checks(q, k, v, positions, freqs, q_weight, k_weight, axes, norm, k_pages, v_pages, slots)
    tokens, heads, d = qh
    qs0, qs1, qs2 = q.stride()
    ks0, ks1, ks2 = k.stride()
    if q_out is None:
        q_out = torch.empty_like(q, memory_format=_CONTIGUOUS)
        os0, os1 = heads * d, d
    else:
        _out_check("q_out", q_out, q, k=k, v=v, k_pages=k_pages, v_pages=v_pages)
        os0, os1, _ = q_out.stride()
    vs0 = vs1 = vs2 = ko0 = ko1 = v_ptr = ko_ptr = pages_ptr = slots_ptr = 0
    if v is not None:
        vs0, vs1, vs2 = v.stride()
        pages = N.Pages(k_pages.data_ptr(), v_pages.data_ptr(), 1, *k_pages.shape, _DTYPES[dt])
        v_ptr, pages_ptr, slots_ptr = v.data_ptr(), ctypes.addressof(pages), slots.data_ptr()
    else:
        if k_out is None:
            k_out = torch.empty_like(k, memory_format=_CONTIGUOUS)
            ko0, ko1 = kh[1] * d, d
        else:
            _out_check("k_out", k_out, k, q=q, q_out=None if q_out is q else q_out)
            ko0, ko1, _ = k_out.stride()
        ko_ptr = k_out.data_ptr()
    if d > 1 and (qs2 != 1 or ks2 != 1 or (v is not None and vs2 != 1)):
        raise ValueError("q, k and v must be [tokens][heads][head_dim] with contiguous head_dim")
    if tokens == 1:  # a dimension of one element may have any stride
        qs0 = ks0 = vs0 = os0 = ko0 = 0
    if heads == 1:
        qs1 = os1 = 0
    if kh[1] == 1:
        ks1 = vs1 = ko1 = 0
    a = tuple(axes) + (0,) * (4 - n_axes)
    status = _entry("oasis_qk_norm_rope")(_ROPE.pack(
        q.data_ptr(), k.data_ptr(), v_ptr, q_out.data_ptr(), ko_ptr, qs0, qs1, ks0, ks1, vs0, vs1, os0, os1, ko0, ko1,
        tokens, heads, kh[1], d, _DTYPES[dt], bool(norm), bool(interleaved), eps,
        0 if q_weight is None else q_weight.data_ptr(), 0 if k_weight is None else k_weight.data_ptr(),
        positions.data_ptr(), pt is torch.int64, freqs.data_ptr(), n_axes, *a, pages_ptr, slots_ptr), _raw_stream(dev))
    if status:
        N.check(status)
    return q_out, k_out


def qk_norm_rope(q: torch.Tensor, k: torch.Tensor, positions: torch.Tensor, freqs: torch.Tensor, *,
                 axes: Sequence[int], interleaved: bool = True, norm: bool = True,
                 q_weight: Optional[torch.Tensor] = None, k_weight: Optional[torch.Tensor] = None,
                 eps: float = 1e-6, q_out: Optional[torch.Tensor] = None,
                 k_out: Optional[torch.Tensor] = None, stream=None) -> Tuple[torch.Tensor, torch.Tensor]:
    """Per-head RMS norm (unless ``norm=False``) and rotation of q [tokens][heads][head_dim] and
    k [tokens][kv_heads][head_dim], bf16, fp16 or fp32, any token and head strides of 16 bytes
    (see ``oasis_qk_norm_rope``).  ``axes`` gives the dims each position axis rotates (their sum
    may be less than head_dim: the rest is only normed), ``positions`` [tokens][len(axes)] int32 or
    int64, ``freqs`` the fp64 frequencies of the pairs (:func:`rope_axis_freqs`).  Pairs are
    neighbours (``interleaved``, as the model here rotates) or halves of the rotated dims.  q_out / k_out may
    be q / k, and otherwise overlap no tensor of the call.  Returns (q_out, k_out)."""
    if stream is not None or q.get_device() != _current_device():
        there = _elsewhere(q.device, stream)
        if there is not None:
            with there:
                return qk_norm_rope(q, k, positions, freqs, axes=axes, interleaved=interleaved, norm=norm,
                                    q_weight=q_weight, k_weight=k_weight, eps=eps, q_out=q_out, k_out=k_out)
    return _rope(q, k, None, positions, freqs, None, None, None, axes, interleaved, norm, q_weight, k_weight, eps,
                 q_out, k_out)


def qk_norm_rope_append(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, positions: torch.Tensor,
                        freqs: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor,
                        slots: torch.Tensor, *, axes: Sequence[int], interleaved: bool = True,
                        norm: bool = True, q_weight: Optional[torch.Tensor] = None,
                        k_weight: Optional[torch.Tensor] = None, eps: float = 1e-6,
                        q_out: Optional[torch.Tensor] = None, stream=None) -> torch.Tensor:
    """:func:`qk_norm_rope` whose keys go, with the values v [tokens][kv_heads][head_dim], into
    cache pages [pages][kv_heads][page_tokens][head_dim]: token i into slot ``slots[i] = page *
    page_tokens + offset`` (int32; a token whose slot lies outside the pages, such as -1, is not stored;
    slots are distinct).  Returns q_out."""
    if stream is not None or q.get_device() != _current_device():
        there = _elsewhere(q.device, stream)
        if there is not None:
            with there:
                return qk_norm_rope_append(q, k, v, positions, freqs, k_pages, v_pages, slots, axes=axes,
                                           interleaved=interleaved, norm=norm, q_weight=q_weight,
                                           k_weight=k_weight, eps=eps, q_out=q_out)
    return _rope(q, k, v, positions, freqs, k_pages, v_pages, slots, axes, interleaved, norm, q_weight, k_weight,
                 eps, q_out, None)[0]


def _attn_checks(q, k_pages, v_pages, page_table, kv_len, cu_q, window, sinks, frame_tokens) -> None:
    _heads3("q", q)
    _cuda("q", q)
    dev = q.device
    tokens, heads, d = q.shape
    _pages(k_pages, v_pages, (4,))
    _cuda("k_pages", k_pages, dev)
    _cuda("v_pages", v_pages, dev)
    if k_pages.shape[3] != d or k_pages.dtype != q.dtype:
        raise ValueError("the pages do not fit the queries (head_dim, type)")
    if page_table.dim() != 2:
        raise ValueError("page_table must be [sequences][pages]")
    batch, width = page_table.shape
    _index32("page_table", page_table, (batch, width), dev)
    _index32("kv_len", kv_len, (batch,), dev)
    if cu_q is not None:
        _index32("cu_q", cu_q, (batch + 1,), dev)
    elif tokens != batch:
        raise ValueError("without cu_q there is one query per sequence")
    if window is not None and window < 1:
        raise ValueError("window must be at least one frame (None: no window)")
    if sinks < 0 or frame_tokens < 1:
        raise ValueError("sinks must be >= 0 and frame_tokens >= 1")
    _no_grad(q, k_pages, v_pages)


def attn_window(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, page_table: torch.Tensor,
                kv_len: torch.Tensor, cu_q: Optional[torch.Tensor] = None, *, window: Optional[int] = None,
                sinks: int = 0, frame_tokens: int = 1, scale: Optional[float] = None,
                max_q: Optional[int] = None, max_kv: Optional[int] = None,
                out: Optional[torch.Tensor] = None, return_lse: bool = False, stream=None):
    """Attention of packed queries over cache pages (see ``oasis_attn_window``).

    q [tokens][heads][head_dim] bf16 or fp16, head_dim 64 or 128; k_pages / v_pages
    [pages][kv_heads][page_tokens][head_dim], heads a multiple of kv_heads, page_tokens of 16.
    Sequence b owns queries ``cu_q[b]:cu_q[b+1]`` (``cu_q`` None: one query each) and ``kv_len[b]``
    cached tokens in the pages ``page_table[b]`` (an entry outside the pages, such as -1, hides its
    tokens); its queries are the last of them.  A query of frame f (``position // frame_tokens``)
    sees the frames up to its own that are fewer than ``window`` frames back (None: all) or among
    the first ``sinks``.  ``scale`` defaults to head_dim ** -0.5.  A query that sees nothing gets zeros.

    ``max_q`` / ``max_kv`` (bounds on the queries and tokens of a sequence) only choose the launch; too
    small ones cost time, and so does a missing ``max_q`` of a batch (all queries count as one sequence's).
    Rows that belong to no sequence are not written.  ``out`` may be q, and otherwise overlaps no tensor of the
    call.  Returns out, or (out, lse)
    with lse fp32 [tokens][heads], the natural logarithm of the softmax sum."""
    dev = q.get_device()
    if stream is not None or dev != _current_device():
        there = _elsewhere(q.device, stream)
        if there is not None:
            with there:
                return attn_window(q, k_pages, v_pages, page_table, kv_len, cu_q, window=window, sinks=sinks,
                                   frame_tokens=frame_tokens, scale=scale, max_q=max_q, max_kv=max_kv, out=out,
                                   return_lse=return_lse)
    qh, gh, th, dt = q.shape, k_pages.shape, page_table.shape, q.dtype
    if not (dev >= 0 and dev == k_pages.get_device() == v_pages.get_device() == page_table.get_device()
            == kv_len.get_device() and len(qh) == 3 and len(gh) == 4 and gh == v_pages.shape and gh[3] == qh[2]
            and dt == k_pages.dtype == v_pages.dtype and (dt is torch.bfloat16 or dt is torch.float16)
            and len(th) == 2 and page_table.dtype is kv_len.dtype is torch.int32 and kv_len.shape == th[:1]
            and k_pages.is_contiguous() and v_pages.is_contiguous() and page_table.is_contiguous()
            and kv_len.is_contiguous() and q.stride(2) == 1
            and (qh[0] == th[0] if cu_q is None else cu_q.get_device() == dev and cu_q.dtype is torch.int32
                 and cu_q.shape == (th[0] + 1,) and cu_q.is_contiguous())
            and (window is None or window >= 1) and sinks >= 0 and frame_tokens >= 1
            and not (q.requires_grad or k_pages.requires_grad or v_pages.requires_grad or _dual_level())):
        _attn_checks(q, k_pages, v_pages, page_table, kv_len, cu_q, window, sinks, frame_tokens)
    tokens, heads, d = qh
    qs0, qs1, _ = q.stride()
    if out is None:
        out = torch.empty_like(q, memory_format=_CONTIGUOUS)
        os0, os1 = heads * d, d
    else:
        _out_check("out", out, q, k_pages=k_pages, v_pages=v_pages)
        os0, os1, _ = out.stride()
    if tokens == 1:  # a dimension of one element may have any stride
        qs0 = os0 = 0
    if heads == 1:
        qs1 = os1 = 0
    lse = torch.empty((tokens, heads), dtype=torch.float32, device=q.device) if return_lse else None
    status = _entry("oasis_attn_window")(_ATTN.pack(
        q.data_ptr(), out.data_ptr(), 0 if lse is None else lse.data_ptr(), qs0, qs1, os0, os1, k_pages.data_ptr(),
        v_pages.data_ptr(), *gh, _DTYPES[dt], page_table.data_ptr(), th[1], kv_len.data_ptr(),
        0 if cu_q is None else cu_q.data_ptr(), th[0], tokens, heads, min(max_q or 0, _BIG), min(max_kv or 0, _BIG),
        min(window or 0, _BIG), min(sinks, _BIG), min(frame_tokens, _BIG), d ** -0.5 if scale is None else scale),
        _raw_stream(dev))
    if status:
        N.check(status)
    return (out, lse) if return_lse else out


_int32_p = ctypes.POINTER(ctypes.c_int32)


def _page_list(name: str, x):
    """(an object that keeps the list, its address, its length) of int32 page numbers."""
    if isinstance(x, torch.Tensor):
        if x.is_cuda:
            raise ValueError(f"{name} must be on the host: it is checked before the launch")
        if x.dtype is torch.int32 and x.dim() == 1 and x.is_contiguous():
            return x, x.data_ptr(), x.numel()
        x = x.numpy()
    x = np.asarray(x)
    if x.size == 0:
        x = x.astype(np.int32)
    if x.ndim != 1 or x.dtype.kind not in "iu":
        raise ValueError(f"{name} must be a list of page numbers")
    if x.dtype != np.int32:
        if x.size and (int(x.max()) > 0x7fffffff or int(x.min()) < 0):
            raise ValueError(f"{name}: page number out of range")
        x = x.astype(np.int32)
    x = np.ascontiguousarray(x)
    return x, x.ctypes.data, x.shape[0]


def copy_pages(k_pages: torch.Tensor, v_pages: torch.Tensor, src, dst, *, to=None, stream=None) -> None:
    """Copy page ``src[i]`` to page ``dst[i]`` for every layer, keys and values, in one launch
    (see ``oasis_pages_copy``).  k_pages / v_pages [(layers)][pages][kv_heads][page_tokens][head_dim];
    ``src`` and ``dst`` are host lists (or int tensors, arrays) of page numbers, free to change once the call returns.
    A page may be copied to several places; within one cache no destination may also be a source.  ``to``:
    the (k, v) pages of another cache that receives the pages."""
    dev, kh, dt = k_pages.get_device(), k_pages.shape, k_pages.dtype
    if stream is not None or dev != _current_device():
        there = _elsewhere(k_pages.device, stream)
        if there is not None:
            with there:
                return copy_pages(k_pages, v_pages, src, dst, to=to)
    if not (dev >= 0 and dev == v_pages.get_device() and kh == v_pages.shape and dt == v_pages.dtype
            and 4 <= len(kh) <= 5 and (dt is torch.bfloat16 or dt is torch.float16)
            and k_pages.is_contiguous() and v_pages.is_contiguous()
            and not (k_pages.requires_grad or v_pages.requires_grad or _dual_level())):
        _cuda("k_pages", k_pages)
        _cuda("v_pages", v_pages, k_pages.device)
        _pages(k_pages, v_pages, (4, 5))
        _no_grad(k_pages, v_pages)
    if to is not None:
        k2, v2 = to
        _pages(k2, v2, (4, 5))
        _cuda("to", k2, k_pages.device)
        _cuda("to", v2, k_pages.device)
        if k2.dim() != len(kh) or k2.dtype != dt or k2.shape[-3:] != kh[-3:] or k2.shape[:-4] != kh[:-4]:
            raise ValueError("the caches' pages differ")
        _no_grad(k2, v2)
    src, src_ptr, n = _page_list("src", src)
    dst, dst_ptr, m = _page_list("dst", dst)
    if n != m:
        raise ValueError("src and dst must have the same length")
    layers = kh[0] if len(kh) == 5 else 1
    a = N.Pages(k_pages.data_ptr(), v_pages.data_ptr(), layers, *kh[-4:], _DTYPES[dt])
    b = a if to is None else N.Pages(k2.data_ptr(), v2.data_ptr(), layers, *k2.shape[-4:], _DTYPES[dt])
    status = N.lib().oasis_pages_copy(a, b, ctypes.cast(src_ptr, _int32_p), ctypes.cast(dst_ptr, _int32_p), n,
                                      _raw_stream(dev))
    if status:
        N.check(status)


class PagedBatchB200:
    """One step of some sessions: their new tokens and where those live in the cache.

    ``cu_q`` int32 [n+1], ``kv_len`` int32 [n], ``page_table`` int32 [n][width], ``slots`` int32
    [tokens]: the device arrays that :func:`attn_window` and :func:`qk_norm_rope_append` take, parts
    of one buffer.  ``max_q``, ``max_kv`` are the launch bounds.  Rebuilt in place by
    ``PagedKVCacheB200.step(..., into=batch)`` (the same sessions' count and tokens), so a captured
    graph that reads it can be replayed step after step."""

    def __init__(self, sequences: int, tokens: int, width: int, page_tokens: int, device):
        self.sequences, self.tokens, self.width = sequences, tokens, width
        self.max_kv = width * page_tokens
        self.max_q = 0
        self.seqs: Tuple[int, ...] = ()
        self.stale = True
        self.cache: Optional[weakref.ref] = None  # whose pages it names
        n = 2 * sequences + 1 + sequences * width + tokens
        self._buffer = torch.empty(n, dtype=torch.int32, device=device)
        cu, lens, table, slots = self._buffer.split([sequences + 1, sequences, sequences * width, tokens])
        self.cu_q, self.kv_len, self.page_table, self.slots = cu, lens, table.view(sequences, width), slots


class _Stream:
    """Host record of a session: its pages in order (-1: evicted), its tokens, and how far pages went
    under each (window, sinks, frame_tokens) of its evictions (a page number, exclusive)."""

    __slots__ = ("pages", "length", "batches", "gone")

    def __init__(self, pages: List[int], length: int, gone: Optional[Dict[Tuple[int, int, int], int]] = None):
        self.pages, self.length = pages, length
        self.batches: List[weakref.ref] = []
        self.gone = dict(gone or {})

    def changed(self) -> None:
        """The plans made of this record no longer describe it."""
        for r in self.batches:
            b = r()
            if b is not None:
                b.stale = True
        self.batches.clear()


class PagedKVCacheB200:
    """K/V pages of any number of sessions, for ``layers`` layers:
    ``k``, ``v`` [layers][pages][kv_heads][page_tokens][head_dim].

    The book is kept on the host; device work is the page copies of :meth:`step` (copy on write),
    :meth:`compact` and :meth:`adopt`, on the current stream.  A method that raises has changed nothing."""

    def __init__(self, layers: int, pages: int, page_tokens: int = 16, kv_heads: int = HEADS,
                 head_dim: int = HEAD_DIM, dtype: torch.dtype = torch.bfloat16, device="cuda"):
        if min(layers, pages, page_tokens, kv_heads) < 1:
            raise ValueError("layers, pages, page_tokens and kv_heads must be positive")
        if page_tokens % 16 or head_dim not in (64, 128) or dtype not in (torch.bfloat16, torch.float16):
            raise ValueError("page_tokens must be a multiple of 16, head_dim 64 or 128, dtype bf16 or fp16")
        if pages * page_tokens > 0x7fffffff:
            raise ValueError("more than 2^31 - 1 token slots")
        self.layers, self.pages, self.page_tokens = layers, pages, page_tokens
        self.kv_heads, self.head_dim, self.dtype = kv_heads, head_dim, dtype
        shape = (layers, pages, kv_heads, page_tokens, head_dim)
        self.k = torch.zeros(shape, dtype=dtype, device=device)
        self.v = torch.zeros(shape, dtype=dtype, device=device)
        self.device = self.k.device
        self._free = list(range(pages - 1, -1, -1))
        self._refs = [0] * pages
        self._seqs: Dict[int, _Stream] = {}
        self._next = 0

    # -- the book ------------------------------------------------------------------------
    def _get(self, seq: int) -> _Stream:
        s = self._seqs.get(seq)
        if s is None:
            raise ValueError(f"no session {seq} in this cache")
        return s

    def _put(self, s: _Stream) -> int:
        seq, self._next = self._next, self._next + 1
        self._seqs[seq] = s
        return seq

    def _drop(self, page: int) -> None:
        if page < 0:
            return
        self._refs[page] -= 1
        if self._refs[page] == 0:
            self._free.append(page)

    def _take(self) -> int:
        page = self._free.pop()
        self._refs[page] = 1
        return page

    @property
    def free_pages(self) -> int:
        return len(self._free)

    @property
    def sessions(self) -> List[int]:
        return list(self._seqs)

    def length(self, seq: int) -> int:
        """Tokens of a session, evicted ones included."""
        return self._get(seq).length

    def pages_of(self, seq: int) -> List[int]:
        """The session's pages in order; -1 where evicted."""
        return list(self._get(seq).pages)

    def new(self) -> int:
        """A new, empty session."""
        return self._put(_Stream([], 0))

    def fork(self, seq: int, copies: int = 1) -> List[int]:
        """``copies`` new sessions that continue ``seq``: they share its pages, and whoever writes
        into a shared page first gets a copy of it.  No device work.  Plans that write into ``seq`` are
        out of date from here on: their slots are shared now."""
        s = self._get(seq)
        copies = operator.index(copies)
        if copies < 0:
            raise ValueError("copies must be >= 0")
        if copies:
            s.changed()
        for p in s.pages:
            if p >= 0:
                self._refs[p] += copies
        return [self._put(_Stream(list(s.pages), s.length, s.gone)) for _ in range(copies)]

    def free(self, seq: int) -> None:
        """End a session; pages that no other session shares become free."""
        s = self._get(seq)
        for p in s.pages:
            self._drop(p)
        s.changed()
        del self._seqs[seq]

    def truncate(self, seq: int, length: int) -> None:
        """Keep the first ``length`` tokens (rejected frames go).  Evicted pages stay evicted; a step whose
        tokens see them is refused."""
        s = self._get(seq)
        if not 0 <= length <= s.length:
            raise ValueError(f"length must be 0..{s.length}")
        keep = -(-length // self.page_tokens)
        for p in s.pages[keep:]:
            self._drop(p)
        del s.pages[keep:]
        s.gone = {w: min(end, keep) for w, end in s.gone.items() if min(end, keep) > self._sink_pages(*w[1:])}
        s.length = length
        s.changed()

    def evict(self, seq: int, window: int, sinks: int = 0, frame_tokens: int = 1) -> int:
        """Give up the pages that no later token of the session can see under this window: all
        their tokens are before the window of the next token's frame and behind the sink frames.
        Returns how many.  Tokens of an earlier frame, written anew, would see them: such a step is
        refused (so evict after the newest frame's last rewrite).  Attention under a wider window does
        not see what has gone."""
        s = self._get(seq)
        if window < 1 or sinks < 0 or frame_tokens < 1:
            raise ValueError("window and frame_tokens must be >= 1, sinks >= 0")
        start = max(0, s.length // frame_tokens - window + 1) * frame_tokens
        end = start // self.page_tokens
        gone = [i for i in range(self._sink_pages(sinks, frame_tokens), end) if s.pages[i] >= 0]
        for i in gone:
            self._drop(s.pages[i])
            s.pages[i] = -1
        if gone:
            w = (window, sinks, frame_tokens)
            s.gone[w] = max(end, s.gone.get(w, 0))
            s.changed()
        return len(gone)

    def _sink_pages(self, sinks: int, frame_tokens: int) -> int:
        """Pages that the sink frames reach into."""
        return -(-sinks * frame_tokens // self.page_tokens)

    # -- device work ---------------------------------------------------------------------
    def copy_pages(self, src, dst, stream=None) -> None:
        """Raw page copies (the book is not touched): see :func:`copy_pages`."""
        copy_pages(self.k, self.v, src, dst, stream=stream)

    def _own(self, wants: Sequence[Tuple[_Stream, int, int]]) -> Tuple[List[List[int]], List[int], List[int], int]:
        """For every (session, first, length): its pages when those of tokens first..length-1 exist and
        belong to the session alone, shared ones that hold tokens to keep copied.  Returns the page lists, the
        copies (sources, destinations) and how many free pages that takes; changes nothing."""
        pt = self.page_tokens
        refs = dict()  # what the references will be: a shared page's last sharer writes in place
        src, dst, taken = [], [], 0
        lists: List[List[int]] = []
        for s, first, length in wants:
            shared = []
            if first < length:
                for (window, _, frame), end in s.gone.items():
                    if (first // frame - window + 1) * frame < end * pt:
                        raise ValueError(f"token {first} sees an evicted page: its session was evicted under a window "
                                         f"of {window} frames of {frame} for later frames")
                for i in range(first // pt, min(-(-length // pt), len(s.pages))):
                    p = s.pages[i]
                    if p < 0:
                        raise ValueError("a token to be written lies in an evicted page")
                    if refs.setdefault(p, self._refs[p]) > 1:
                        refs[p] -= 1
                        shared.append(i)
            pages = list(s.pages)
            new = len(shared) + max(0, -(-length // pt) - len(pages))
            free = self._free[max(0, len(self._free) - taken - new): len(self._free) - taken][::-1]  # as _take will
            taken += new
            if taken <= len(self._free):
                for i, p in zip(shared, free):
                    src.append(pages[i])
                    dst.append(p)
                    pages[i] = p
                pages.extend(free[len(shared):])
            lists.append(pages)
        if taken > len(self._free):
            raise RuntimeError(f"paged KV cache: {taken} pages needed, {len(self._free)} free")
        return lists, src, dst, taken

    def step(self, seqs: Sequence[int], tokens: Union[int, Sequence[int]], *, extend: bool = True,
             table_width: Optional[int] = None, into: Optional[PagedBatchB200] = None,
             stream=None) -> PagedBatchB200:
        """The plan of one step: ``tokens`` new tokens for each session (one number or one each).
        With ``extend=False`` the step's tokens are the sessions' last ones again (the same frame
        at another solver step: its keys and values are written anew).  Pages are taken, and
        shared ones that the step writes into are copied first.  ``table_width``: pages per session
        the plan has room for (default: what this step needs).  ``into``: rebuild this plan in place, on ``stream``
        (default: the current one), for the same number of sessions and tokens.  A new plan's memory belongs to
        that stream."""
        seqs = [int(i) for i in seqs]
        if not seqs or len(set(seqs)) != len(seqs):
            raise ValueError("a step takes one or more different sessions")
        counts = [int(tokens)] * len(seqs) if isinstance(tokens, (int, np.integer)) else [int(t) for t in tokens]
        if len(counts) != len(seqs) or min(counts) < 0:
            raise ValueError("one token count >= 0 per session")
        streams = [self._get(i) for i in seqs]
        lengths = [s.length + (n if extend else 0) for s, n in zip(streams, counts)]
        if any(n > m for n, m in zip(counts, lengths)):
            raise ValueError("a session has fewer tokens than the step rewrites")
        pt, total = self.page_tokens, sum(counts)
        need = max(1, max(-(-m // pt) for m in lengths))
        width = into.width if into is not None else max(need, table_width or 0)
        if need > width:
            raise ValueError(f"the plan has room for {width} pages per session, {need} are needed")
        if into is not None and into.cache is not None and into.cache() is not self:
            raise ValueError("the plan is of another cache")
        if into is not None and (into.sequences != len(seqs) or into.tokens != total):
            raise ValueError(f"the plan is for {into.sequences} sessions and {into.tokens} tokens")
        if width * pt > 0x3fffffff:
            raise ValueError("more than 2^30 - 1 tokens in a session")
        # everything that can fail comes before the book changes
        lists, src, dst, taken = self._own([(s, m - n, m) for s, n, m in zip(streams, counts, lengths)])
        n = len(seqs)
        host = np.full(2 * n + 1 + n * width + total, -1, np.int32)
        cu = host[: n + 1]
        cu[0] = 0
        np.cumsum(counts, out=cu[1:])
        host[n + 1: 2 * n + 1] = lengths
        table = host[2 * n + 1: 2 * n + 1 + n * width].reshape(n, width)
        slots = host[2 * n + 1 + n * width:]
        for i, (pages, c, m) in enumerate(zip(lists, counts, lengths)):
            table[i, : len(pages)] = pages
            at = np.arange(m - c, m)
            slots[cu[i]: cu[i + 1]] = table[i, at // pt].astype(np.int64) * pt + at % pt
        with _elsewhere(self.device, stream) or contextlib.nullcontext():  # a new plan's memory is the stream's, too
            b = into if into is not None else PagedBatchB200(n, total, width, pt, self.device)
            if src:
                self.copy_pages(src, dst)
            b._buffer.copy_(torch.from_numpy(host))
        for _ in range(taken):
            self._take()
        for p in src:
            self._drop(p)
        for s, pages, m in zip(streams, lists, lengths):
            if m != s.length or pages != s.pages:
                s.pages, s.length = pages, m
                s.changed()
        b.max_q = max(max(counts), b.max_q)  # a captured launch keeps the bound it was captured with
        b.cache = weakref.ref(self)
        for i in b.seqs:  # a rebuilt plan no longer follows its earlier sessions
            old = self._seqs.get(i)
            if old is not None:
                old.batches = [r for r in old.batches if r() is not b]
        b.seqs, b.stale = tuple(seqs), False
        for s in streams:
            s.batches = [r for r in s.batches if r() is not None] + [weakref.ref(b)]
        return b

    def compact(self, stream=None) -> int:
        """Move the used pages to the front of the pools (one launch) and return their number."""
        used = self.pages - len(self._free)
        src = [p for p in range(used, self.pages) if self._refs[p]]
        dst = [p for p in range(used) if not self._refs[p]]
        if src:
            self.copy_pages(src, dst, stream)
            to = dict(zip(src, dst))
            for s in self._seqs.values():
                s.pages = [to.get(p, p) for p in s.pages]
                s.changed()
            for p, n in to.items():
                self._refs[n], self._refs[p] = self._refs[p], 0
        self._free = list(range(self.pages - 1, used - 1, -1))
        return used

    def adopt(self, other: "PagedKVCacheB200", seq: int, stream=None) -> int:
        """A session of another cache (of the same layers, heads, page size and type) continues here:
        its pages are copied, sharing is not kept.  Returns its number here; the other keeps its own."""
        if other is self:
            raise ValueError("adopt takes a session of another cache: fork one of this")
        for name in ("layers", "page_tokens", "kv_heads", "head_dim", "dtype", "device"):
            if getattr(other, name) != getattr(self, name):
                raise ValueError(f"the caches differ in {name}")
        s = other._get(seq)
        held = [p for p in s.pages if p >= 0]
        if len(held) > len(self._free):
            raise RuntimeError(f"paged KV cache: {len(held)} pages needed, {len(self._free)} free")
        dst = self._free[len(self._free) - len(held):][::-1]
        if held:
            copy_pages(other.k, other.v, held, dst, to=(self.k, self.v), stream=stream)
        taken = iter([self._take() for _ in held])
        return self._put(_Stream([next(taken) if p >= 0 else -1 for p in s.pages], s.length, s.gone))

    # -- a layer's operators on a step -----------------------------------------------------
    def _live(self, batch: PagedBatchB200) -> None:
        if batch.cache is None or batch.cache() is not self:
            raise ValueError("the plan is of another cache")
        if batch.stale:
            raise ValueError("the step's plan is out of date: its sessions' pages have changed since")

    def append(self, layer: int, batch: PagedBatchB200, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
               positions: torch.Tensor, freqs: torch.Tensor, **kw) -> torch.Tensor:
        """:func:`qk_norm_rope_append` of the step's tokens into this layer's pages."""
        self._live(batch)
        return qk_norm_rope_append(q, k, v, positions, freqs, self.k[layer], self.v[layer], batch.slots, **kw)

    def attend(self, layer: int, batch: PagedBatchB200, q: torch.Tensor, **kw):
        """:func:`attn_window` of the step's queries over this layer's pages."""
        self._live(batch)
        return attn_window(q, self.k[layer], self.v[layer], batch.page_table, batch.kv_len, batch.cu_q,
                           max_q=max(1, batch.max_q), max_kv=batch.max_kv, **kw)
