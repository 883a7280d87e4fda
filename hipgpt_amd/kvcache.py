"""Paged key/value cache in 8 bits over libhipgpt_attn.so (``include/hipgpt_attn.h``).

HipGPT keeps no cache (its generation loop recomputes the window,
``src/gpt_model.cpp:261-273``); :func:`hipgpt_amd.attention.decode_kvcache` keeps a
contiguous fp32 one.  Here keys and values live in pages of 32, 64 or 128 tokens as
8-bit codes with one scale per (page, head), query heads may share cached heads, and
sequences of a batch bring ragged chunks of new tokens.

* :class:`CacheQ8` -- the pools of one layer.
* :class:`Batch` -- one step's sequences (pages, lengths, new tokens), for all layers.
* :func:`append` -- rotate q and k by position, quantise k and v into the pages.
* :func:`read` -- the values that cached tokens stand for.
* :func:`decode` -- one query row per sequence, split over the keys.
* :func:`prefill` -- a chunk of new tokens per sequence, causal.
* :func:`rope_freqs` -- the rotation's frequencies.

A step, in every layer: ``q = append(cache, batch, q, k, v, freqs=f)`` (``advance=True``
in the first), then ``decode`` or ``prefill`` on that ``q``.  Nothing synchronises with
the host; lengths and page tables are read on the device.
"""
from __future__ import annotations

import ctypes
import functools

import torch

from . import _lib
from .attention import _need_cuda, _ptr

_TYPES = {torch.float32: _lib.F32, torch.bfloat16: _lib.BF16}
# the stream handle alone: torch.cuda.current_stream() builds an object around it, 2.7 us a call
_raw_stream = torch._C._cuda_getCurrentRawStream
_current_device = torch._C._cuda_getDevice


def _dtype(name, t):
    dt = _TYPES.get(t.dtype)
    if dt is None:
        raise TypeError(f"{name} must be float32 or bfloat16")
    return dt


def _tensor(name, t):
    if not isinstance(t, torch.Tensor) or t.dim() != 3:
        raise ValueError(f"{name} must be a [rows, heads, D] tensor")
    return t


class CacheQ8:
    """Pools of one layer: ``k``, ``v`` uint8 [pages, heads, page_size, D] (the last two
    dims contiguous; v's bytes are in the tile order of the header), ``k_scale``,
    ``v_scale`` float32 [pages, heads]."""

    def __init__(self, k, v, k_scale, v_scale):
        for name, t, dt in (("k", k, torch.uint8), ("v", v, torch.uint8), ("k_scale", k_scale, torch.float32),
                            ("v_scale", v_scale, torch.float32)):
            _need_cuda(name, t, dt)
            if t.device != k.device:
                raise ValueError("the pools must be on one device")
        if k.dim() != 4 or v.shape != k.shape or v.stride() != k.stride():
            raise ValueError("k, v must be [pages, heads, page_size, D] with the same strides")
        P, H, ps, D = k.shape
        if k.stride(3) != 1 or k.stride(2) != D:
            raise ValueError("each (page, head) of k, v must be contiguous")
        if tuple(k_scale.shape) != (P, H) or v_scale.shape != k_scale.shape or v_scale.stride() != k_scale.stride():
            raise ValueError("k_scale, v_scale must be [pages, heads] with the same strides")
        self.k, self.v, self.k_scale, self.v_scale = k, v, k_scale, v_scale
        self.device, self.heads, self.page_size, self.head_dim = k.device, H, ps, D
        self.index = k.device.index
        self._c = _lib.KvQ8Cache(k.data_ptr(), v.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(),
                                 k.stride(0), k.stride(1), k_scale.stride(0), k_scale.stride(1), P, ps, H, D)
        self._ref = ctypes.byref(self._c)

    @classmethod
    def empty(cls, pages, heads, page_size, head_dim, device="cuda"):
        """Pools without content (a page's scale is set by its first token)."""
        codes = torch.empty(2, pages, heads, page_size, head_dim, dtype=torch.uint8, device=device)
        scales = torch.empty(2, pages, heads, dtype=torch.float32, device=device)
        return cls(codes[0], codes[1], scales[0], scales[1])


class Batch:
    """One step's sequences: ``block_table`` int32 [B, max_pages], ``lens`` int32 [B]
    (tokens with the step's new ones), ``cu_new`` int32 [B + 1] (rows of the new tokens;
    None: one each, row b), all on the device.  ``max_new``: the most new tokens of a
    sequence; ``max_len``: a bound of ``lens`` that the default split goes by."""

    def __init__(self, block_table, lens, cu_new=None, max_new=1, max_len=None):
        _need_cuda("block_table", block_table, torch.int32)
        _need_cuda("lens", lens, torch.int32)
        if block_table.dim() != 2 or (block_table.shape[1] > 1 and block_table.stride(1) != 1):
            raise ValueError("block_table must be [B, max_pages] with contiguous rows")
        B, M = block_table.shape
        if tuple(lens.shape) != (B,) or not lens.is_contiguous() or lens.device != block_table.device:
            raise ValueError("lens must be a contiguous int32 tensor of B elements beside block_table")
        if cu_new is not None:
            _need_cuda("cu_new", cu_new, torch.int32)
            if tuple(cu_new.shape) != (B + 1,) or not cu_new.is_contiguous() or cu_new.device != lens.device:
                raise ValueError("cu_new must be a contiguous int32 tensor of B + 1 elements beside block_table")
        elif max_new != 1:
            raise ValueError("max_new is 1 without cu_new")
        self.block_table, self.lens, self.cu_new = block_table, lens, cu_new  # kept alive
        self.device, self.size, self.max_new = lens.device, B, int(max_new)
        self.max_len = None if max_len is None else int(max_len)
        self._c = _lib.KvQ8Batch(block_table.data_ptr(), block_table.stride(0), lens.data_ptr(), _ptr(cu_new), B, M,
                                 self.max_new)
        self._ref = ctypes.byref(self._c)

    def capacity(self, cache):
        """The most tokens a sequence's row of the table can hold."""
        return self._c.max_pages * cache.page_size


def rope_freqs(rot_dim, base=10000.0, device="cuda"):
    """Turns per position of the ``rot_dim / 2`` rotated pairs as 0.64 fixed point
    (int64 tensor), for :func:`append`."""
    f = (ctypes.c_uint64 * max(1, rot_dim // 2))()
    _lib.check(_lib.lib().hipgpt_rope_freqs(f, rot_dim, float(base)), "hipgpt_rope_freqs")
    return torch.tensor(list(f), dtype=torch.int64, device=device)


def _rows(name, t, shape, dtype, device):
    """(token, head) strides of a tensor of that shape with contiguous D."""
    if not isinstance(t, torch.Tensor) or t.device != device:
        raise TypeError(f"{name} must be a tensor on {device}")
    if t.dtype is not dtype:
        raise TypeError(f"{name} must be {dtype}, got {t.dtype}")
    st = t.stride()
    if t.shape != shape or st[2] != 1:
        raise ValueError(f"{name} must be {list(shape)} with contiguous D")
    return st[:2]


def _enter(cache, batch):
    """None where the cache's device is current, else a context that makes it so."""
    if batch.device != cache.device:
        raise ValueError("cache and batch must be on one device")
    return None if _current_device() == cache.index else torch.cuda.device(cache.device)


def _handle(cache, stream, *owned):
    """Handle of the stream to launch on.  ``owned``: tensors allocated here, on the current
    stream, that another stream's kernels will use."""
    if stream is None:
        return _raw_stream(cache.index)
    for t in owned:
        if t is not None:
            t.record_stream(stream)
    return stream.cuda_stream


def append(cache, batch, q, k, v, freqs=None, interleaved=False, q_out=None, advance=False, stream=None):
    """Rotates and quantises the new tokens into the cache; returns the rotated q.

    k, v: [T, heads, D], q: [T, Hq, D] or None, all float32 or all bfloat16; ``freqs``:
    :func:`rope_freqs` of the rotated head dims (None: no rotation); ``q_out`` may be q.
    ``advance`` first raises ``batch.lens`` by the new tokens."""
    other = _enter(cache, batch)
    if other is not None:
        with other:
            return append(cache, batch, q, k, v, freqs, interleaved, q_out, advance, stream)
    _tensor("k", k)
    dt, dtype, dev = _dtype("k", k), k.dtype, cache.device
    T, D = k.shape[0], cache.head_dim
    shape = (T, cache.heads, D)
    ks = _rows("k", k, shape, dtype, dev)
    vs = _rows("v", v, shape, dtype, dev)
    Hq, qs, os_, mine, qp, op = 0, (0, 0), (0, 0), None, 0, 0
    if q is not None:
        Hq = _tensor("q", q).shape[1]
        shape = (T, Hq, D)
        qs = _rows("q", q, shape, dtype, dev)
        if q_out is None:
            q_out = mine = torch.empty_like(q)
        os_ = _rows("q_out", q_out, shape, dtype, dev)
        qp, op = q.data_ptr(), q_out.data_ptr()
    elif q_out is not None:
        raise ValueError("q_out without q")
    rot = fp = 0
    if freqs is not None:
        if freqs.dtype is not torch.int64 or freqs.device != dev or freqs.dim() != 1 or not freqs.is_contiguous():
            raise TypeError("freqs must be what rope_freqs gives, on the cache's device")
        rot, fp = 2 * freqs.numel(), freqs.data_ptr()
    rc = _lib.lib().hipgpt_kvq8_append(
        cache._ref, batch._ref, T, qp, op, k.data_ptr(), v.data_ptr(), Hq, *qs, *os_, *ks, *vs, fp, rot,
        1 if interleaved else 0, dt, 1 if advance else 0, _handle(cache, stream, mine))
    if rc:
        _lib.check(rc, "hipgpt_kvq8_append")
    return q_out


def read(cache, batch, T, dtype=torch.float32, k=None, v=None, stream=None):
    """(k, v) [T, heads, D]: the values of each sequence's last ``cu_new[b + 1] -
    cu_new[b]`` tokens, packed in that order (T rows in all)."""
    other = _enter(cache, batch)
    if other is not None:
        with other:
            return read(cache, batch, T, dtype, k, v, stream)
    shape = (T, cache.heads, cache.head_dim)
    mine = [None, None]
    if k is None:
        k = mine[0] = torch.empty(shape, device=cache.device, dtype=dtype if v is None else v.dtype)
    if v is None:
        v = mine[1] = torch.empty(shape, device=cache.device, dtype=k.dtype)
    ks = _rows("k", k, shape, k.dtype, cache.device)
    vs = _rows("v", v, shape, k.dtype, cache.device)
    rc = _lib.lib().hipgpt_kvq8_read(cache._ref, batch._ref, T, k.data_ptr(), v.data_ptr(), *ks, *vs, _dtype("k", k),
                                     _handle(cache, stream, *mine))
    if rc:
        _lib.check(rc, "hipgpt_kvq8_read")
    return k, v


@functools.lru_cache(maxsize=4096)
def default_splits(B, T, max_new, Hq, heads, D, out_dtype, max_len):
    """The split count that the library picks for these sizes."""
    return int(_lib.lib().hipgpt_attn_kvq8_default_splits(B, T, max_new, Hq, heads, D, _TYPES[out_dtype], max_len))


def workspace_bytes(B, T, max_new, Hq, heads, D, out_dtype, num_splits):
    return int(_lib.lib().hipgpt_attn_kvq8_workspace_bytes(B, T, max_new, Hq, heads, D, _TYPES[out_dtype],
                                                           num_splits))


def _attention(name, rows, cache, batch, q, out, out_dtype, scale, num_splits, workspace, stream):
    """Both attention entry points; ``rows``: (T,) where the entry point takes it."""
    other = _enter(cache, batch)
    if other is not None:
        with other:
            return _attention(name, rows, cache, batch, q, out, out_dtype, scale, num_splits, workspace, stream)
    T, Hq, _ = q.shape
    H, D, dev = cache.heads, cache.head_dim, cache.device
    shape = (T, Hq, D)
    dt = _dtype("q", q)
    qs = _rows("q", q, shape, q.dtype, dev)
    mine = [None, None]
    if out is None:
        out = mine[0] = torch.empty(shape, dtype=out_dtype, device=dev)
    os_ = _rows("out", out, shape, out.dtype, dev)
    odt = _dtype("out", out)
    if num_splits is None:
        num_splits = default_splits(batch.size, T, batch.max_new, Hq, H, D, out.dtype,
                                    min(batch.max_len or batch.capacity(cache), 0x7fffffff))
    ns = int(num_splits)
    wp = nbytes = 0
    if ns > 1:
        if workspace is None:
            need = workspace_bytes(batch.size, T, batch.max_new, Hq, H, D, out.dtype, ns)
            workspace = mine[1] = torch.empty(need, dtype=torch.uint8, device=dev)
        elif workspace.device != dev or not workspace.is_contiguous():
            raise ValueError(f"workspace must be contiguous, on {dev}")
        wp, nbytes = workspace.data_ptr(), workspace.numel() * workspace.element_size()
    rc = getattr(_lib.lib(), name)(
        cache._ref, batch._ref, *rows, q.data_ptr(), out.data_ptr(), Hq, *qs, *os_,
        -1.0 if scale is None else float(scale), dt, odt, 1 if ns < 1 else ns, wp, nbytes,
        _handle(cache, stream, *mine))
    if rc:
        _lib.check(rc, name)
    return out


def decode(cache, batch, q, out=None, out_dtype=torch.float32, scale=None, num_splits=None, workspace=None,
           stream=None):
    """softmax(q k^T * scale) v of q [B, Hq, D] over each sequence's cached tokens.

    float32 or bfloat16 q; ``out``: [B, Hq, D] float32, or bfloat16 for a bfloat16 q.
    ``num_splits`` partitions of the work (default: the library's choice for
    ``batch.max_len``); ``workspace``: caller-owned, :func:`workspace_bytes` (allocated
    here if None)."""
    if _tensor("q", q).shape[0] != batch.size:
        raise ValueError("q must have one row per sequence")
    return _attention("hipgpt_attn_decode_kvq8", (), cache, batch, q, out, out_dtype, scale, num_splits, workspace,
                      stream)


def prefill(cache, batch, q, out=None, out_dtype=torch.float32, scale=None, num_splits=None, workspace=None,
            stream=None):
    """Causal attention of each sequence's new tokens (q [T, Hq, D], packed as
    ``batch.cu_new``) over its cache, which holds them already.  The rest as
    :func:`decode`."""
    return _attention("hipgpt_attn_prefill_kvq8", (_tensor("q", q).shape[0],), cache, batch, q, out, out_dtype, scale,
                      num_splits, workspace, stream)
