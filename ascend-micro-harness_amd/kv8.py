"""The 8-bit paged KV cache over libtq4.so (include/tq4_kv8.h).

A serving step is four calls: `paged_plan` makes the block tables and the slot
map from the requests' lengths, on the GPU; `kv8_reshape_and_cache` writes the
step's keys and values; `kv8_paged_decode` (one row a sequence) or
`kv8_paged_prefill` (several) attends. `kv8_cache` allocates a pool.

The cache's element type is the tensors': torch.float8_e4m3fn or torch.int8,
with one FP32 scale for each (page, head) of the keys and of the values. The
step's activations are BF16 or FP16; their rows may lie apart (slices of one
projection's output), each row contiguous.

As in the other entry points, a refused call raises ValueError before anything
is launched, and calls run on the current stream (or `stream`). Tensors lie on
one GPU, which need not be the current one. What a call allocates (`out`,
`workspace`) belongs to the stream that it runs on.
"""
from __future__ import annotations

import contextlib
import ctypes as C
import math

import torch

from . import tq4 as _tq4
from .tq4 import _P, _check, _done, _need, _ptr

KV8_FP8 = torch.float8_e4m3fn
KV8_INT8 = torch.int8
KV8_MAX_SPLITS = 256
_U32, _U64, _F32, _I32, _SZ = C.c_uint32, C.c_uint64, C.c_float, C.c_int, C.c_size_t
_CODES = {KV8_FP8: 0, KV8_INT8: 1}
_ELEMENTS = {torch.float16: 0, torch.bfloat16: 1}
_INT = (torch.int32,)

_bound = None


def _lib():
    global _bound
    if _bound is None:
        L = _tq4.lib()
        L.tq4_paged_plan_workspace_bytes.restype = _SZ
        L.tq4_paged_plan_workspace_bytes.argtypes = [_U32]
        L.tq4_paged_plan.restype = _I32
        L.tq4_paged_plan.argtypes = [_P] * 14 + [_SZ] + [_U32] * 5
        L.tq4_kv8_reshape_and_cache.restype = _I32
        L.tq4_kv8_reshape_and_cache.argtypes = [_P, _I32, _I32] + [_P] * 6 + [_U64] * 2 + [_U32] * 5
        L.tq4_kv8_decode_workspace_bytes.restype = _SZ
        L.tq4_kv8_decode_workspace_bytes.argtypes = [_U32] * 7
        L.tq4_kv8_paged_decode.restype = _I32
        L.tq4_kv8_paged_decode.argtypes = ([_P, _I32, _I32] + [_P] * 7 + [_SZ, _P, _U64] +
                                           [_U32] * 8 + [_F32])
        L.tq4_kv8_prefill_workspace_bytes.restype = _SZ
        L.tq4_kv8_prefill_workspace_bytes.argtypes = [_U32] * 8
        L.tq4_kv8_paged_prefill.restype = _I32
        L.tq4_kv8_paged_prefill.argtypes = ([_P, _I32, _I32] + [_P] * 8 + [_SZ, _P, _U64] +
                                            [_U32] * 9 + [_I32, _F32])
        _bound = L
    return _bound


def _fast():
    """The native checks (csrc/tq4_host.cpp) where they are in use."""
    if _bound is None:
        _lib()
    return _tq4._fast


@contextlib.contextmanager
def _on(device, stream):
    """The device and stream of a call, and the stream's handle."""
    with torch.cuda.device(device):
        s = torch.cuda.current_stream() if stream is None else stream
        if s.device != device:
            raise ValueError(f"the stream is on {s.device}, the tensors on {device}")
        with torch.cuda.stream(s):
            yield _P(s.cuda_stream)


def _one_device(what, first, tensors):
    """Every tensor on the first one's GPU."""
    name0, t0 = first
    if not t0.is_cuda:
        raise ValueError(f"{name0} must be a device tensor")
    for name, t in tensors:
        if t is None:
            continue
        if not t.is_cuda:
            raise ValueError(f"{name} must be a device tensor")
        if t.device != t0.device:
            raise ValueError(f"{what}: {name} is on {t.device}, {name0} on {t0.device}")


def _sizes(what, **sizes):
    """Sizes that the C ABI's 32 bits hold (ctypes would cut the others to them)."""
    for name, n in sizes.items():
        if not 0 <= n < 1 << 32:
            raise ValueError(f"{what}: {name} must lie in [0, 2^32), got {n}")


def _rows(what, name, t):
    """Activations [rows][heads][d], each row contiguous: the row stride in elements."""
    _need(what, name, t, tuple(_ELEMENTS), ndim=3)
    n, heads, d = t.shape
    inner = (heads <= 1 or t.stride(1) == d) and (d <= 1 or t.stride(2) == 1)
    if not inner or (n > 1 and t.stride(0) < heads * d):
        raise ValueError(f"{what}: the rows of {name} must be contiguous [heads][head_size] and "
                         f"lie apart, got strides {tuple(t.stride())}")
    return t.stride(0) if n > 1 else heads * d


def _pool(what, key_cache, value_cache, scale_cache):
    """(num_blocks, num_kv_heads, block_size, head_size) of a cache."""
    _need(what, "key_cache", key_cache, tuple(_CODES), ndim=4)
    _need(what, "value_cache", value_cache, (key_cache.dtype,), numel=key_cache.numel())
    P, H, S, d = key_cache.shape
    _need(what, "scale_cache", scale_cache, (torch.float32,), numel=2 * P * H)
    return P, H, S, d


def kv8_cache(num_blocks, num_kv_heads, block_size, head_size, dtype=KV8_FP8, device="cuda"):
    """A zeroed pool: key_cache [P][H][S][d], value_cache [P][H][S/16][d][16]
    and scale_cache [2][P][H] (FP32)."""
    if dtype not in _CODES:
        raise ValueError(f"kv8_cache: dtype must be float8_e4m3fn or int8, got {dtype}")
    if block_size <= 0 or block_size % 16:
        raise ValueError(f"kv8_cache: block_size must be a multiple of 16, got {block_size}")
    n = (num_blocks, num_kv_heads, block_size, head_size)
    key = torch.zeros(n, dtype=torch.uint8, device=device).view(dtype)
    value = torch.zeros((num_blocks, num_kv_heads, block_size // 16, head_size, 16),
                        dtype=torch.uint8, device=device).view(dtype)
    return key, value, torch.zeros((2, num_blocks, num_kv_heads), device=device)


# ------------------------------------------------------------------- the plan
def paged_plan(context_lens, query_lens, block_tables, free_pages, free_state, slot_mapping,
               cu_seqlens, granted, block_size, release=None, positions=None,
               new_context_lens=None, new_free_state=None, workspace=None, stream=None):
    """Block tables, slot map and positions of a step from the requests'
    lengths (tq4_paged_plan). All tensors int32: context_lens, query_lens,
    granted and release [B], block_tables [B][max_blocks], free_pages [P] (the
    ring of free pages), free_state {head, count}, slot_mapping and positions
    [rows], cu_seqlens [B + 1]. new_context_lens and new_free_state None: in
    place. The table entries of a released context and the ring's free entries
    all have to name pages: one that names none is handed on like a page."""
    what = "paged_plan"
    f = _fast()
    if f is not None and _done(f.paged_plan(
            context_lens, query_lens, block_tables, free_pages, free_state, slot_mapping,
            cu_seqlens, granted, block_size, release, positions, new_context_lens, new_free_state,
            workspace, stream), what):
        return
    _sizes(what, block_size=block_size)
    _need(what, "block_tables", block_tables, _INT, ndim=2)
    B, M = block_tables.shape
    _need(what, "context_lens", context_lens, _INT, numel=B)
    _need(what, "query_lens", query_lens, _INT, numel=B)
    _need(what, "free_pages", free_pages, _INT, min_numel=1)
    _need(what, "free_state", free_state, _INT, numel=2)
    _need(what, "slot_mapping", slot_mapping, _INT)
    _need(what, "cu_seqlens", cu_seqlens, _INT, numel=B + 1)
    _need(what, "granted", granted, _INT, numel=B)
    _need(what, "release", release, _INT, numel=B, optional=True)
    _need(what, "positions", positions, _INT, numel=slot_mapping.numel(), optional=True)
    _need(what, "new_context_lens", new_context_lens, _INT, numel=B, optional=True)
    _need(what, "new_free_state", new_free_state, _INT, numel=2, optional=True)
    _one_device(what, ("block_tables", block_tables),
                (("context_lens", context_lens), ("query_lens", query_lens),
                 ("free_pages", free_pages), ("free_state", free_state),
                 ("slot_mapping", slot_mapping), ("cu_seqlens", cu_seqlens), ("granted", granted),
                 ("release", release), ("positions", positions),
                 ("new_context_lens", new_context_lens), ("new_free_state", new_free_state),
                 ("workspace", workspace)))
    if new_context_lens is None:
        new_context_lens = context_lens
    if new_free_state is None:
        new_free_state = free_state
    with _on(block_tables.device, stream) as st:
        if workspace is None:
            workspace = torch.empty(int(_lib().tq4_paged_plan_workspace_bytes(B)),
                                    dtype=torch.uint8, device=block_tables.device)
        _check(_lib().tq4_paged_plan(
            st, _ptr(context_lens), _ptr(query_lens), _ptr(release), _ptr(block_tables),
            _ptr(free_pages), _ptr(free_state), _ptr(slot_mapping), _ptr(positions),
            _ptr(cu_seqlens), _ptr(granted), _ptr(new_context_lens), _ptr(new_free_state),
            _ptr(workspace), workspace.numel() * workspace.element_size(), B, M, block_size,
            free_pages.numel(), slot_mapping.numel()), what)


# ----------------------------------------------------------------- the writer
def kv8_reshape_and_cache(key, value, key_cache, value_cache, scale_cache, slot_mapping,
                          stream=None):
    """BF16 or FP16 keys and values [tokens][kv_heads][d] into the cache at
    slot_mapping (int32, page * block_size + offset; others write nothing)."""
    what = "kv8_reshape_and_cache"
    f = _fast()
    if f is not None and _done(f.kv8_reshape_and_cache(key, value, key_cache, value_cache,
                                                       scale_cache, slot_mapping, stream), what):
        return
    ks = _rows(what, "key", key)
    _need(what, "value", value, (key.dtype,), ndim=3)
    if value.shape != key.shape:
        raise ValueError(f"{what}: value must have key's shape, got {tuple(value.shape)}")
    vs = _rows(what, "value", value)
    P, H, S, d = _pool(what, key_cache, value_cache, scale_cache)
    T = key.shape[0]
    if tuple(key.shape[1:]) != (H, d):
        raise ValueError(f"{what}: key has rows {tuple(key.shape[1:])}, the cache {(H, d)}")
    _need(what, "slot_mapping", slot_mapping, _INT, min_numel=T)
    _one_device(what, ("key", key), (("value", value), ("key_cache", key_cache),
                                     ("value_cache", value_cache), ("scale_cache", scale_cache),
                                     ("slot_mapping", slot_mapping)))
    if T == 0:
        return
    with _on(key.device, stream) as st:
        _check(_lib().tq4_kv8_reshape_and_cache(
            st, _ELEMENTS[key.dtype], _CODES[key_cache.dtype], _P(key.data_ptr()),
            _P(value.data_ptr()), _ptr(key_cache), _ptr(value_cache), _ptr(scale_cache),
            _ptr(slot_mapping), ks, vs, T, H, d, S, P), what)


# -------------------------------------------------------------- the attention
def _attention_args(what, q, key_cache, value_cache, scale_cache, block_tables, context_lens,
                    out, workspace, more=(), one_row=False):
    stride = _rows(what, "q", q)
    P, H, S, d = _pool(what, key_cache, value_cache, scale_cache)
    if q.shape[2] != d:
        raise ValueError(f"{what}: q has head size {q.shape[2]}, the cache {d}")
    _need(what, "block_tables", block_tables, _INT, ndim=2)
    B, M = block_tables.shape
    if one_row and q.shape[0] != B:
        raise ValueError(f"{what}: {q.shape[0]} rows of q for {B} sequences")
    _need(what, "context_lens", context_lens, _INT, numel=B)
    _need(what, "out", out, (q.dtype,), numel=q.numel(), optional=True)
    _one_device(what, ("q", q), (("key_cache", key_cache), ("value_cache", value_cache),
                                 ("scale_cache", scale_cache), ("block_tables", block_tables),
                                 ("context_lens", context_lens), ("out", out),
                                 ("workspace", workspace)) + tuple(more))
    return stride, P, H, S, d, B, M


def _room(nbytes, workspace, device):
    if workspace is None and nbytes:
        workspace = torch.empty(nbytes, dtype=torch.uint8, device=device)
    return workspace, workspace.numel() * workspace.element_size() if workspace is not None else 0


def kv8_decode_workspace_bytes(num_seqs, num_heads, num_kv_heads, head_size, block_size,
                               max_blocks_per_seq, num_splits=0):
    """Bytes of workspace that kv8_paged_decode needs (0: none); any contents."""
    _sizes("kv8_decode_workspace_bytes", num_seqs=num_seqs, num_heads=num_heads,
           num_kv_heads=num_kv_heads, head_size=head_size, block_size=block_size,
           max_blocks_per_seq=max_blocks_per_seq, num_splits=num_splits)
    return int(_lib().tq4_kv8_decode_workspace_bytes(num_seqs, num_heads, num_kv_heads, head_size,
                                                     block_size, max_blocks_per_seq, num_splits))


def kv8_paged_decode(q, key_cache, value_cache, scale_cache, block_tables, context_lens, out=None,
                     workspace=None, num_splits=0, scale=None, stream=None):
    """softmax(scale * q . k) v for one row a sequence: q [B][heads][d] BF16 or
    FP16 -> out, of q's type, contiguous. scale None: 1 / sqrt(d). workspace
    None: allocated where one is needed (kv8_decode_workspace_bytes)."""
    what = "kv8_paged_decode"
    f = _fast()
    if f is not None:
        r = f.kv8_paged_decode(q, key_cache, value_cache, scale_cache, block_tables, context_lens,
                               out, workspace, num_splits, scale, stream)
        if _done(r, what):
            return r
    stride, P, H, S, d, B, M = _attention_args(what, q, key_cache, value_cache, scale_cache,
                                               block_tables, context_lens, out, workspace,
                                               one_row=True)
    Hq = q.shape[1]
    if not 0 <= num_splits <= KV8_MAX_SPLITS:
        raise ValueError(f"{what}: num_splits must be 0 (auto) to {KV8_MAX_SPLITS}, got {num_splits}")
    if scale is None:
        scale = 1.0 / math.sqrt(d)
    with _on(q.device, stream) as st:
        if out is None:
            out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
        ws, nbytes = _room(kv8_decode_workspace_bytes(B, Hq, H, d, S, M, num_splits), workspace,
                           q.device)
        _check(_lib().tq4_kv8_paged_decode(
            st, _ELEMENTS[q.dtype], _CODES[key_cache.dtype], _P(q.data_ptr()), _ptr(key_cache),
            _ptr(value_cache), _ptr(scale_cache), _ptr(block_tables), _ptr(context_lens), _ptr(ws),
            nbytes, _ptr(out), stride, B, Hq, H, d, S, P, M, num_splits, scale), what)
    return out


def kv8_prefill_workspace_bytes(num_rows, num_seqs, num_heads, num_kv_heads, head_size,
                                block_size, max_blocks_per_seq, max_query_len):
    """Bytes of workspace that kv8_paged_prefill needs (0: none); any contents."""
    max_query_len = min(max_query_len, num_rows)
    _sizes("kv8_prefill_workspace_bytes", num_rows=num_rows, num_seqs=num_seqs,
           num_heads=num_heads, num_kv_heads=num_kv_heads, head_size=head_size,
           block_size=block_size, max_blocks_per_seq=max_blocks_per_seq,
           max_query_len=max_query_len)
    return int(_lib().tq4_kv8_prefill_workspace_bytes(num_rows, num_seqs, num_heads, num_kv_heads,
                                                      head_size, block_size, max_blocks_per_seq,
                                                      max_query_len))


def kv8_paged_prefill(q, key_cache, value_cache, scale_cache, block_tables, context_lens,
                      cu_seqlens, max_query_len, causal=True, out=None, workspace=None, scale=None,
                      stream=None):
    """softmax(scale * q . k) v for several rows a sequence: q [rows][heads][d],
    sequence b's rows cu_seqlens[b] .. cu_seqlens[b + 1], at most max_query_len.
    causal: row i of n sees the tokens up to context_lens[b] - n + i; otherwise
    all of them (cross attention). Rows of no sequence are left as they are in
    `out` (undefined where the call allocates it)."""
    what = "kv8_paged_prefill"
    f = _fast()
    if f is not None:
        r = f.kv8_paged_prefill(q, key_cache, value_cache, scale_cache, block_tables, context_lens,
                                cu_seqlens, max_query_len, causal, out, workspace, scale, stream)
        if _done(r, what):
            return r
    stride, P, H, S, d, B, M = _attention_args(
        what, q, key_cache, value_cache, scale_cache, block_tables, context_lens, out, workspace,
        (("cu_seqlens", cu_seqlens),))
    _need(what, "cu_seqlens", cu_seqlens, _INT, numel=B + 1)
    if max_query_len < 0:
        raise ValueError(f"{what}: max_query_len must not be negative, got {max_query_len}")
    T, Hq = q.shape[:2]
    max_query_len = min(max_query_len, T)
    if scale is None:
        scale = 1.0 / math.sqrt(d)
    with _on(q.device, stream) as st:
        if out is None:
            out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
        ws, nbytes = _room(kv8_prefill_workspace_bytes(T, B, Hq, H, d, S, M, max_query_len),
                           workspace, q.device)
        _check(_lib().tq4_kv8_paged_prefill(
            st, _ELEMENTS[q.dtype], _CODES[key_cache.dtype], _P(q.data_ptr()), _ptr(key_cache),
            _ptr(value_cache), _ptr(scale_cache), _ptr(block_tables), _ptr(context_lens),
            _ptr(cu_seqlens), _ptr(ws), nbytes, _ptr(out), stride, T, B, Hq, H, d, S, P, M,
            max_query_len, bool(causal), scale), what)
    return out


__all__ = ["KV8_FP8", "KV8_INT8", "KV8_MAX_SPLITS", "kv8_cache", "paged_plan",
           "kv8_reshape_and_cache", "kv8_decode_workspace_bytes", "kv8_paged_decode",
           "kv8_prefill_workspace_bytes", "kv8_paged_prefill"]
