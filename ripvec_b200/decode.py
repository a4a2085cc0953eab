"""Decoder-side operators over a paged key/value cache (torch device tensors).

What runs after a search: a decoder reads the retrieved text, either as one prefix that a batch of
answers shares or as the candidates of a rerank batch behind one query.  ``PagedCache`` describes one
layer's pools, ``DecodeStep`` plans a step once for all layers and runs ``append`` (rotary positions,
keys and values into their pages) and ``attend`` (attention of every sequence over its group's shared
prefix and its own keys), and ``rms_norm`` is the decoder's residual norm with 16-bit or 8-bit output.

Calls queue their kernels on ``stream`` (a CUDA stream handle; by default torch's current stream) and
return.  An output that a call makes itself is memory of that stream, as of a tensor made under
``torch.cuda.stream``; tensors of other streams are the caller's to order and to keep until the work is done
(``record_stream``).  The reference has no decoder; there is nothing of it to cite here.
"""

from __future__ import annotations

import ctypes as C
from itertools import chain
from struct import Struct
from typing import Sequence

import numpy as np
import torch

from . import _lib as L

_DTYPES = {torch.bfloat16: L.RV_DTYPE_BF16, torch.float16: L.RV_DTYPE_F16}


# The calls' arguments as one record each (``rv_step_append_args`` and so on): packing 17 arguments and passing one
# pointer takes 0.4 us on the host, converting 17 arguments 2.3 us.
_append_args = Struct("P" + "Pqq" * 4 + "PPqiiP").pack
_attend_args = Struct("P" + "Pqq" * 2 + "PdP").pack
_norm_args = Struct("PqPqPPqPqPqiiiidiP").pack

# torch's current stream of a device as a handle, without the stream object around it.
_current_stream = torch._C._cuda_getCurrentRawStream


def _new(stream: int | None, like, shape: tuple, strides: tuple, dtype=None):
    """A tensor for ``stream`` to write.  torch's allocator hands out memory in the order of the stream that is
    current: on another one an earlier owner's reads could still be to come."""
    if stream is None or stream == _current_stream(like.get_device()):
        return like.new_empty_strided(shape, strides, dtype=dtype)
    # (0 and 1, cudaStreamLegacy, are the default stream.)
    other = torch.cuda.ExternalStream(stream, like.device) if stream > 1 else torch.cuda.default_stream(like.device)
    with torch.cuda.stream(other):
        return like.new_empty_strided(shape, strides, dtype=dtype)


def _rows(name: str, t, shape: tuple, cache: "PagedCache") -> tuple:
    """Address, token stride and head stride of ``t``, which must be ``shape`` rows like the cache's."""
    try:
        st, sh, sd = t.stride()
    except ValueError:  # not of 3 axes
        sd = st = sh = 0
    if sd != 1 or t.shape != shape or t.dtype is not cache.dtype or t.get_device() != cache.device_index:
        raise ValueError(f"{name} must be {shape} {cache.dtype} on {cache.device} with unit stride along the last "
                         f"axis, got {tuple(t.shape)} {t.dtype} on {t.device} with strides {t.stride()}")
    return t.data_ptr(), st, sh


def _i32(values) -> np.ndarray:
    a = np.asarray(values)
    if a.size and (a.dtype.kind not in "iu" or a.min() < 0 or a.max() > np.iinfo(np.int32).max):
        raise ValueError("lengths, sizes and pages are whole numbers from 0 to 2^31 - 1")
    return np.ascontiguousarray(a, np.int32)


class PagedCache:
    """One layer's key and value pools, ``[pages, kv_heads, page_size, head_dim]`` bf16 or f16 tensors in
    any order of memory (pass a transposed view of other layouts) with unit stride along ``head_dim`` and
    the same strides.  The tensors are the caller's and are kept alive by this object."""

    def __init__(self, k: torch.Tensor, v: torch.Tensor):
        if k.ndim != 4 or k.shape != v.shape or k.dtype not in _DTYPES or v.dtype != k.dtype or not k.is_cuda \
                or v.device != k.device:
            raise ValueError("k and v must be 4-D bf16 or f16 tensors of one shape on one CUDA device")
        if k.stride() != v.stride() or k.stride(3) != 1:
            raise ValueError("k and v must have the same strides, and unit stride along the last axis")
        self.k, self.v = k, v
        self.num_pages, self.kv_heads, self.page_size, self.head_dim = k.shape
        self.dtype, self.device, self.device_index = k.dtype, k.device, k.get_device()
        sp, sh, ss, _ = k.stride()
        self.desc = L.KvCache(k.data_ptr(), v.data_ptr(), self.num_pages, sp, sh, ss, _DTYPES[k.dtype], self.kv_heads,
                              self.head_dim, self.page_size)
        self._ref = C.addressof(self.desc)


class DecodeStep:
    """A step of a batch: planned once on the host, then run by every layer (``rv_step_*``)."""

    def __init__(self, *, q_heads: int, kv_heads: int, head_dim: int, page_size: int, device: int = 0):
        self._lib = L.lib()
        h = C.c_void_p()
        rc = self._lib.rv_step_create(device, q_heads, kv_heads, head_dim, page_size, C.byref(h))
        if rc != L.RV_OK:
            raise L.RvError(rc, "rv_step_create failed (q_heads a multiple of kv_heads, head_dim 64 or 128, page_size "
                                "16, 32, 64, 128 or 256, a CUDA device)")
        self._h = h
        self.q_heads, self.kv_heads, self.head_dim, self.page_size = q_heads, kv_heads, head_dim, page_size
        self.device = torch.device("cuda", device)
        self.tokens = None  # of the plan; None without one

    def _check(self, rc: int) -> None:
        if rc != L.RV_OK:
            raise L.RvError(rc, self._lib.rv_step_last_error(self._h).decode())

    def _tokens(self, cache: PagedCache) -> int:
        if self.tokens is None:
            raise L.RvError(L.RV_E_NOT_READY, "no plan")
        if cache.device_index != self.device.index:
            raise ValueError(f"the cache's device {cache.device} is not the step's, {self.device}")
        return self.tokens

    def close(self) -> None:
        if getattr(self, "_h", None):
            self._lib.rv_step_destroy(self._h)
            self._h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def plan(self, *, q_lens: Sequence[int], own_lens: Sequence[int], own_pages: Sequence[Sequence[int]],
             num_pages: int, prefix_lens: Sequence[int] = (), prefix_pages: Sequence[Sequence[int]] = (),
             group_sizes: Sequence[int] | None = None, causal: bool = True, stream: int | None = None) -> None:
        """``rv_step_plan``: sequence ``b`` brings ``q_lens[b]`` new tokens and has ``own_lens[b]`` keys of
        its own, these included, in ``own_pages[b]`` (longer lists are cut; a padded 2-D numpy table will do
        and is the quickest).  Consecutive sequences form groups that share a prefix; by default one group
        of all, with no prefix or the one given."""
        self.tokens = None
        ps = self.page_size
        ql, ol, pl = _i32(q_lens), _i32(own_lens), _i32(prefix_lens)
        if len(ql) != len(ol) or len(own_pages) != len(ol) or len(prefix_pages) != len(pl):
            raise ValueError("q_lens, own_lens and own_pages (and prefix_lens and prefix_pages) must have equal lengths")
        if group_sizes is None:
            if len(pl) > 1:
                raise ValueError("several prefixes need group_sizes")
            gs = _i32([len(ql)])
            if len(pl) == 0:
                pl, prefix_pages = _i32([0]), [[]]
        else:
            gs = _i32(group_sizes)
            if len(gs) != len(pl):
                raise ValueError("group_sizes and prefix_lens must have equal lengths")

        def flat(lists, lens):
            need = -(-lens.astype(np.int64) // ps)
            if isinstance(lists, np.ndarray) and lists.ndim == 2:  # a page table, padded rows
                if len(need) and need.max() > lists.shape[1]:
                    raise ValueError("a page list is shorter than its length needs")
                return _i32(lists[np.arange(lists.shape[1]) < need[:, None]])
            need = need.tolist()
            if any(len(p) < k for p, k in zip(lists, need)):
                raise ValueError("a page list is shorter than its length needs")
            kept = (p if len(p) == k else p[:k] for p, k in zip(lists, need))
            return _i32(np.fromiter(chain.from_iterable(kept), np.int64, sum(need)))

        op, pp = flat(own_pages, ol), flat(prefix_pages, pl)
        self._check(self._lib.rv_step_plan(self._h, len(ql), ql.ctypes.data, ol.ctypes.data, op.ctypes.data, len(gs),
                                           gs.ctypes.data, pl.ctypes.data, pp.ctypes.data, num_pages, bool(causal),
                                           _current_stream(self.device.index) if stream is None else stream))
        self.tokens = int(ql.sum())

    def append(self, cache: PagedCache, q, k, v, cos, sin, *, q_out=None, interleaved: bool = False,
               stream: int | None = None):
        """``rv_step_append``: rotates ``q [tokens, q_heads, head_dim]`` and ``k [tokens, kv_heads, head_dim]``
        by ``cos`` / ``sin [positions, rot / 2]`` (f32) and writes keys and values into the cache; returns
        the rotated queries (``q_out``, a new tensor by default; it may be ``q``).  ``q = None`` appends
        keys and values only."""
        t, d = self._tokens(cache), self.head_dim
        if q is not None:
            qa = _rows("q", q, (t, self.q_heads, d), cache)
            if q_out is None:
                q_out = _new(stream, q, (t, self.q_heads, d), (self.q_heads * d, d, 1))
            qo = _rows("q_out", q_out, (t, self.q_heads, d), cache)
        elif q_out is not None:
            raise ValueError("q_out without q")
        else:
            qa = qo = (0, 0, 0)
        ka, va = _rows("k", k, (t, self.kv_heads, d), cache), _rows("v", v, (t, self.kv_heads, d), cache)
        if cos.ndim != 2 or cos.shape != sin.shape or cos.dtype is not torch.float32 or sin.dtype is not torch.float32 \
                or cos.get_device() != cache.device_index or sin.get_device() != cache.device_index \
                or not cos.is_contiguous() or not sin.is_contiguous():
            raise ValueError("cos and sin must be contiguous [positions, rot / 2] f32 tensors on the cache's device")
        positions, half = cos.shape
        rc = self._lib.rv_step_append_record(self._h, _append_args(
            cache._ref, *qa, *ka, *va, *qo, cos.data_ptr(), sin.data_ptr(), positions, 2 * half, interleaved,
            _current_stream(cache.device_index) if stream is None else stream))
        if rc:
            self._check(rc)
        return q_out

    def attend(self, cache: PagedCache, q, *, out=None, lse=None, scale: float | None = None,
               stream: int | None = None):
        """``rv_step_attend``: attention of every query of the step over its group's prefix and its own keys
        (``scale`` 1 / sqrt(head_dim) by default).  ``lse [tokens, q_heads]`` f32, where given, receives the
        log of the softmax's denominator.  Returns ``out [tokens, q_heads, head_dim]``."""
        t, d = self._tokens(cache), self.head_dim
        shape = (t, self.q_heads, d)
        qa = _rows("q", q, shape, cache)
        if out is None:
            out = _new(stream, q, shape, (self.q_heads * d, d, 1))
        oa = _rows("out", out, shape, cache)
        if lse is not None and (lse.shape != shape[:2] or lse.dtype is not torch.float32
                                or lse.get_device() != cache.device_index or not lse.is_contiguous()):
            raise ValueError(f"lse must be a contiguous [{t}, {self.q_heads}] f32 tensor on the cache's device")
        rc = self._lib.rv_step_attend_record(self._h, _attend_args(
            cache._ref, *qa, *oa, 0 if lse is None else lse.data_ptr(), d ** -0.5 if scale is None else scale,
            _current_stream(cache.device_index) if stream is None else stream))
        if rc:
            self._check(rc)
        return out


def rms_norm(x, weight, *, residual=None, residual_out=None, out=None, eps: float = 1e-5, out_8bit: bool = False,
             group: int = 0, scales=None, stream: int | None = None):
    """``rv_rms_norm`` over the rows of ``x [rows, hidden]`` (bf16 or f16, ``weight`` f32): ``h = x + residual``,
    ``out = h / sqrt(mean(h^2) + eps) * weight``; ``h`` in 16 bits goes to ``residual_out`` where given (it may
    be ``residual`` or ``x``).  Returns ``(out, scales)``: 16-bit rows and ``None``, or with ``out_8bit`` e4m3
    codes and their f32 scales ``[rows, hidden / group]`` (``group = 0``: one scale a row)."""
    dtype, dev, shape = x.dtype, x.get_device(), x.shape
    code = _DTYPES.get(dtype)
    if code is None or dev < 0 or len(shape) != 2:
        raise ValueError("x must be a 2-D bf16 or f16 CUDA tensor")
    rows, hidden = shape
    xs, unit = x.stride()
    rp = rs = rop = ros = 0
    if residual is not None:
        rp, (rs, u) = residual.data_ptr(), residual.stride()
        if residual.shape != shape or residual.dtype is not dtype or residual.get_device() != dev or u != 1 < hidden:
            raise ValueError("residual must be like x, with unit stride along the last axis")
    if residual_out is not None:
        rop, (ros, u) = residual_out.data_ptr(), residual_out.stride()
        if residual_out.shape != shape or residual_out.dtype is not dtype or residual_out.get_device() != dev \
                or u != 1 < hidden:
            raise ValueError("residual_out must be like x, with unit stride along the last axis")
    if unit != 1 < hidden:
        raise ValueError("x must have unit stride along the last axis")
    if weight.shape != shape[1:] or weight.dtype is not torch.float32 or weight.get_device() != dev \
            or not weight.is_contiguous():
        raise ValueError("weight must be a contiguous f32 [hidden] tensor on x's device")
    if out_8bit:
        if group and (group not in (32, 64, 128, 256) or hidden % group):
            raise ValueError("group must be 32, 64, 128 or 256 and divide hidden")
        dtype, code_out = torch.float8_e4m3fn, L.RV_DTYPE_E4M3
        per_row = hidden // group if group else 1
        if scales is None:
            scales = _new(stream, weight, (rows, per_row), (per_row, 1))
        elif scales.shape != (rows, per_row) or scales.dtype is not torch.float32 or scales.get_device() != dev \
                or not scales.is_contiguous():
            raise ValueError(f"scales must be a contiguous {(rows, per_row)} f32 tensor on x's device")
        sp = scales.data_ptr()
    else:
        if group or scales is not None:
            raise ValueError("group and scales come with out_8bit")
        code_out, sp = code, 0
    if out is None:
        out = _new(stream, x, shape, (hidden, 1), dtype)
        os = hidden
    else:
        os, u = out.stride()
        if out.shape != shape or out.dtype is not dtype or out.get_device() != dev or u != 1 < hidden:
            raise ValueError(f"out must be {tuple(shape)} {dtype} on x's device, with unit stride along the last axis")
    if rows == 0:
        return out, scales
    rc = L.lib().rv_rms_norm_record(_norm_args(
        x.data_ptr(), xs, rp, rs, weight.data_ptr(), rop, ros, out.data_ptr(), os, sp, rows, hidden, code, code_out, group,
        eps, dev, _current_stream(dev) if stream is None else stream))
    if rc:
        raise L.RvError(rc, "rv_rms_norm failed (hidden from 1 to 65536, row strides of at least hidden, eps >= 0)")
    return out, scales
