"""Paged K/V cache of grouped heads on MI355X: rows written into it, read back, and
decode attention over it (bf16, or fp8 with one scale for each token and head).

The reference has no counterpart: its decode ops are the absorbed-MLA ones
(moonmath reference moonmath_attention/mla.py:41-186). These serve models with
ordinary (grouped, multi- or single-head) keys and values.

A cache is a pair ``k_cache`` / ``v_cache`` of shape [num_blocks, Hkv, page, D],
bfloat16 or float8_e4m3fn, D 64, 128 or 256, page a power of two of at least 16
tokens. Only the last dim has to be contiguous (rows on 16-byte boundaries), so
a token-major cache [num_blocks, page, Hkv, D] is passed as its
``transpose(1, 2)``, and K and V may be slices of one tensor. An fp8 cache comes
with ``k_scale`` / ``v_scale``, float32 [num_blocks, Hkv, page] (last dim
contiguous, rows on 16-byte boundaries): the row of a token and head stands for
its codes times its scale.

Every op runs on the caller's current stream without a host synchronisation and
can be captured into a graph; lengths, tables and slots are read on the device.
"""
import ctypes
import math

import torch

from . import _checks as ck
from . import _lib

__all__ = ["gqa_decode_paged", "gqa_kv_read", "gqa_kv_write"]

_FP8 = torch.float8_e4m3fn
_DIMS = (64, 128, 256)
_MAX_Q_LEN = 8
_MAX_HEADS = 1 << 16
_MAX_TOKENS = (1 << 31) - 4096
_MAX_ROW_STRIDE = 1 << 26


def _check_cache(k_cache, v_cache, k_scale, v_scale, who, written):
    """(num_blocks, Hkv, page, D, fp8) of a cache."""
    if not isinstance(k_cache, torch.Tensor) or not isinstance(v_cache, torch.Tensor):
        raise TypeError(f"{who}: k_cache and v_cache must be torch.Tensor")
    if k_cache.dtype not in (torch.bfloat16, _FP8):
        raise ValueError(f"{who}: k_cache must be bfloat16 or float8_e4m3fn, got {k_cache.dtype}")
    fp8 = k_cache.dtype == _FP8
    if k_cache.dim() != 4 or k_cache.shape[3] not in _DIMS:
        raise ValueError(f"{who}: k_cache must be [num_blocks, Hkv, page, D] with D 64, 128 or 256")
    nb, heads, page, D = k_cache.shape
    if v_cache.shape != k_cache.shape:
        raise ValueError(f"{who}: v_cache's shape {list(v_cache.shape)} must be k_cache's {list(k_cache.shape)}")
    if nb < 1 or heads < 1:
        raise ValueError(f"{who}: the cache must hold at least one block and head")
    if page < 16 or page & (page - 1):
        raise ValueError(f"{who}: pages must hold a power of two of at least 16 tokens, got {page}")
    if nb * page > 1 << 31:
        raise ValueError(f"{who}: the cache must hold at most 2^31 tokens")
    for name, t in (("k_cache", k_cache), ("v_cache", v_cache)):
        ck.tensor(t, name, who, k_cache.dtype)
        ck.rows(t, name, who)
        if t.stride(2) > _MAX_ROW_STRIDE:
            raise ValueError(f"{who}: {name}'s tokens lie more than 2^26 elements apart")
        if written:
            ck.one_place_each(t, name, who)
    if (k_scale is not None) != fp8 or (v_scale is not None) != fp8:
        raise ValueError(f"{who}: k_scale and v_scale go with a float8_e4m3fn cache, and only with one")
    if fp8:
        for name, t in (("k_scale", k_scale), ("v_scale", v_scale)):
            ck.tensor(t, name, who, torch.float32)
            if t.shape != k_cache.shape[:3]:
                raise ValueError(f"{who}: {name} must be [num_blocks, Hkv, page] = {list(k_cache.shape[:3])}")
            ck.rows(t, name, who)
            if written:
                ck.one_place_each(t, name, who)
    if written and not (ck.share_none(k_cache, v_cache) and (not fp8 or ck.share_none(k_scale, v_scale))):
        raise ValueError(f"{who}: the K and V caches must not share memory")
    return nb, heads, page, D, fp8


def _check_ints(t, name, who):
    if not isinstance(t, torch.Tensor) or t.dtype != torch.int32:
        raise ValueError(f"{who}: {name} must be int32")


def _cache_strides(cache, scale):
    s = cache.stride()
    return [s[0], s[1], s[2]] + ([scale.stride(0), scale.stride(1)] if scale is not None else [0, 0])


def _strides(*values):
    return (ctypes.c_longlong * len(values))(*values)


def _run(fn_name, *args):
    rc = getattr(_lib.lib, fn_name)(*args)
    if rc != 0:
        raise RuntimeError(f"{fn_name} returned error code {rc}")


def _check_rows(k, v, slots, heads, D, who, written):
    for name, t in (("k", k), ("v", v)):
        ck.tensor(t, name, who, torch.bfloat16)
        if t.dim() != 3 or t.shape[1] != heads or t.shape[2] != D:
            raise ValueError(f"{who}: {name} must be [N, {heads}, {D}], got {list(t.shape)}")
        ck.rows(t, name, who)
        if written:
            ck.one_place_each(t, name, who)
    N = k.shape[0]
    if v.shape[0] != N:
        raise ValueError(f"{who}: k and v must hold the same number of tokens")
    if written and not ck.share_none(k, v):
        raise ValueError(f"{who}: k and v are written, and must not share memory")
    if slots.dim() != 1 or slots.shape[0] != N or not slots.is_contiguous():
        raise ValueError(f"{who}: slots must be contiguous with one entry per token ({N}), got {list(slots.shape)}")
    return N


def gqa_kv_write(k, v, k_cache, v_cache, slots, k_scale=None, v_scale=None) -> None:
    """Write new tokens' K and V rows into the cache.

    k, v [N, Hkv, D] bf16 (any strides with a contiguous last dim and rows on
    16-byte boundaries: slices of a fused projection); slots int32 [N]: token i
    goes to row slots[i] % page of block slots[i] // page, in both caches; a
    negative slot (padding token) or one past the cache writes nothing. The
    slots of one call must differ: of two tokens with the same slot, parts of
    either may stay.

    A bf16 cache takes the rows as they are. For an fp8 cache each row (token,
    head) gets scale = max(amax / 448, 2^-126), amax over its finite values, and
    codes e4m3fn(x / scale), rounded to nearest even; a value that is not finite
    becomes NaN. k and v must lie apart from the caches, and the K and V caches
    (and their scales) must not share memory: slices of one tensor are fine.
    """
    if _lib.calls.gqa_write(k, v, k_cache, v_cache, slots, k_scale, v_scale):
        return
    who = "gqa_kv_write"
    nb, heads, page, D, _ = _check_cache(k_cache, v_cache, k_scale, v_scale, who, True)
    _check_ints(slots, "slots", who)
    N = _check_rows(k, v, slots, heads, D, who, False)
    if not all(ck.apart(a, b) for a in (k, v) for b in (k_cache, v_cache)):
        raise ValueError(f"{who}: k and v must lie apart from the caches")
    dev = k.device
    ck.on_device(who, dev, v=v, k_cache=k_cache, v_cache=v_cache, slots=slots, k_scale=k_scale, v_scale=v_scale)
    strides = _strides(*k.stride()[:2], *v.stride()[:2], *_cache_strides(k_cache, k_scale),
                       *_cache_strides(v_cache, v_scale))
    p = _lib.ptr
    with torch.cuda.device(dev):
        _run("launch_gqa_kv_write", p(k), p(v), p(k_cache), p(v_cache), p(k_scale), p(v_scale), p(slots), N, heads, D,
             nb, page, strides, _lib.stream_ptr(dev))


def gqa_kv_read(k_cache, v_cache, slots, k_scale=None, v_scale=None, *, k=None, v=None):
    """Read rows of the cache back: (k, v), bf16 [N, Hkv, D] of the tokens in
    ``slots`` (int32 [N], numbered as in ``gqa_kv_write``; the same slot may
    come twice). An fp8 row is bf16(code * scale), rounded to nearest even. A
    negative slot, or one past the cache, gives a row of zeros. ``k`` and ``v``
    are optional outputs (any strides with a contiguous last dim and rows on
    16-byte boundaries), apart from the caches and sharing no memory.
    """
    res = _lib.calls.gqa_read(k_cache, v_cache, slots, k_scale, v_scale, k, v)
    if res is not None:
        return res
    who = "gqa_kv_read"
    nb, heads, page, D, _ = _check_cache(k_cache, v_cache, k_scale, v_scale, who, False)
    _check_ints(slots, "slots", who)
    if slots.dim() != 1 or not slots.is_contiguous():
        raise ValueError(f"{who}: slots must be contiguous [N]")
    shape = (slots.shape[0], heads, D)
    k = torch.empty(shape, dtype=torch.bfloat16, device=slots.device) if k is None else k
    v = torch.empty(shape, dtype=torch.bfloat16, device=slots.device) if v is None else v
    N = _check_rows(k, v, slots, heads, D, who, True)
    if not all(ck.apart(a, b) for a in (k, v) for b in (k_cache, v_cache)):
        raise ValueError(f"{who}: k and v must lie apart from the caches")
    dev = k_cache.device
    ck.on_device(who, dev, v_cache=v_cache, slots=slots, k_scale=k_scale, v_scale=v_scale, k=k, v=v)
    strides = _strides(*k.stride()[:2], *v.stride()[:2], *_cache_strides(k_cache, k_scale),
                       *_cache_strides(v_cache, v_scale))
    p = _lib.ptr
    with torch.cuda.device(dev):
        _run("launch_gqa_kv_read", p(k_cache), p(v_cache), p(k_scale), p(v_scale), p(slots), p(k), p(v), N, heads, D,
             nb, page, strides, _lib.stream_ptr(dev))
    return k, v


def gqa_decode_paged(q, k_cache, v_cache, seq_lens, block_table, *, scale=None, k_scale=None, v_scale=None, out=None,
                     return_lse=False):
    """Decode attention of each request's last tokens over its pages.

    q [B, Hq, D] (one query) or [B, q_len, Hq, D] (draft window, q_len <= 8) bf16,
    any strides with a contiguous last dim and rows on 16-byte boundaries; query
    head h reads kv head h // (Hq / Hkv). seq_lens int32 [B]: request b's tokens in
    the cache, its queries' own included; block_table int32 [B, max_blocks]: token t
    of request b is row t % page of block block_table[b, t // page]. Query t of q_len
    attends tokens [0, S - q_len + t + 1); scale defaults to 1 / sqrt(D).

    Returns bf16 of q's shape (``out``, if given: q itself, or apart from q), rounded
    to nearest even; with ``return_lse`` also the float32 [B, (q_len,) Hq] ln of the
    softmax's sum, by which outputs over parts of a context join. A query that sees no
    token gives zeros and -inf. Table entries past a request's length are not used,
    and what cache rows past it hold reaches no output; lengths are clamped to
    [0, max_blocks * page], page ids to the cache. Sums of weighted V are held in
    float32 before they are divided by the weights' sum: |V| times the number of
    tokens has to stay below 3.4e38. Calls share nothing: each takes its own
    workspace from torch's allocator.
    """
    res = _lib.calls.gqa_decode(q, k_cache, v_cache, seq_lens, block_table, scale, k_scale, v_scale, out, return_lse)
    if res is not None:
        return res
    who = "gqa_decode_paged"
    nb, heads, page, D, fp8 = _check_cache(k_cache, v_cache, k_scale, v_scale, who, False)
    ck.tensor(q, "q", who, torch.bfloat16)
    if q.dim() not in (3, 4) or q.shape[-1] != D:
        raise ValueError(f"{who}: q must be [B, Hq, {D}] or [B, q_len, Hq, {D}], got {list(q.shape)}")
    ck.rows(q, "q", who)
    q4 = q if q.dim() == 4 else q.unsqueeze(1)
    B, q_len, Hq = q4.shape[:3]
    if not 1 <= q_len <= _MAX_Q_LEN:
        raise ValueError(f"{who}: q_len must be in [1,{_MAX_Q_LEN}]")
    if Hq < 1 or Hq % heads or Hq > _MAX_HEADS:
        raise ValueError(f"{who}: Hq = {Hq} must be a multiple of the cache's {heads} heads, and at most 65536")
    _check_ints(seq_lens, "seq_lens", who)
    _check_ints(block_table, "block_table", who)
    if seq_lens.dim() != 1 or seq_lens.shape[0] != B or not seq_lens.is_contiguous():
        raise ValueError(f"{who}: seq_lens must be contiguous [B] = [{B}], got {list(seq_lens.shape)}")
    if block_table.dim() != 2 or block_table.shape[0] != B or block_table.shape[1] < 1:
        raise ValueError(f"{who}: block_table must be [B, max_blocks] with B = {B}, got {list(block_table.shape)}")
    if block_table.shape[1] * page > _MAX_TOKENS:
        raise ValueError(f"{who}: a request's table must hold at most 2^31 - 4096 tokens")
    if block_table.shape[1] > 1 and block_table.stride(1) != 1:
        raise ValueError(f"{who}: block_table's last dim must be contiguous")
    if out is not None:
        ck.tensor(out, "out", who, torch.bfloat16)
        if out.shape != q.shape:
            raise ValueError(f"{who}: out must have q's shape {list(q.shape)}, got {list(out.shape)}")
        ck.rows(out, "out", who)
        ck.one_place_each(out, "out", who)
        same = out.data_ptr() == q.data_ptr() and out.stride() == q.stride()
        if not (same or ck.apart(out, q)) or not (ck.apart(out, k_cache) and ck.apart(out, v_cache)):
            raise ValueError(f"{who}: out must be q itself or lie apart from it, and apart from the caches")
    scale = 1.0 / math.sqrt(D) if scale is None else float(scale)
    dev = q.device
    ck.on_device(who, dev, k_cache=k_cache, v_cache=v_cache, seq_lens=seq_lens, block_table=block_table,
                 k_scale=k_scale, v_scale=v_scale, out=out)
    if out is None:
        out = torch.empty(q.shape, dtype=q.dtype, device=dev)
    lse = torch.empty(q.shape[:-1], dtype=torch.float32, device=dev) if return_lse else None
    o4 = out if out.dim() == 4 else out.unsqueeze(1)
    width = block_table.shape[1]
    strides = _strides(*q4.stride()[:3], *o4.stride()[:3], *_cache_strides(k_cache, k_scale),
                       *_cache_strides(v_cache, v_scale), block_table.stride(0))
    p = _lib.ptr
    with torch.cuda.device(dev):
        nbytes = _lib.lib.moonmath_gqa_decode_workspace(B, q_len, Hq, heads, D, page, width, int(fp8), strides)
        ws = torch.empty(nbytes, dtype=torch.uint8, device=dev) if nbytes else None
        _run("launch_gqa_decode_paged", p(q), p(k_cache), p(v_cache), p(k_scale), p(v_scale), p(out), p(lse),
             p(seq_lens), p(block_table), B, q_len, Hq, heads, D, nb, page, width, strides, scale, p(ws),
             _lib.stream_ptr(dev))
    return (out, lse) if return_lse else out
