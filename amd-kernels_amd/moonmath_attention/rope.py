"""AxialRope: rotary positions of one or several axes on MI355X.

The reference has no counterpart (its callers rotate q and k themselves before
``forward``, moonmath reference moonmath_attention/_kernel.py:14-82). An image's or
video's tokens have a position on each axis (time, height, width); text tokens are
the case of one axis, or of the same number on each.

Typical use before an attention call::

    rope = moonmath_attention.AxialRope((8, 28, 28))          # pairs per axis: 128 dims
    q, k = rope(q, k, positions, layout="bshd")               # positions int32 [3, S]
    out = moonmath_attention.forward(q, k, v, layout="bshd")
"""
import ctypes
import math

import torch

from . import _checks as ck
from . import _lib

__all__ = ["AxialRope"]

_DIMS = (64, 128, 256)


class AxialRope:
    """Rotates pairs of a head's dims by positions on several axes.

    Args:
        sections: pairs of dims that belong to each axis, in order; their sum P is
            a multiple of 8, and 2P at most the head dim (64, 128 or 256). Dims past
            2P pass through.
        theta: base of the frequencies.
        frequencies: "axis": pair i of an axis's n turns by theta^(-i / n) radians
            for each position, so each axis has the whole range; "shared": pair p of
            all P by theta^(-p / P), and the sections cut one range between the axes.
        pairing: "halves": dims (p, P + p) are a pair; "adjacent": dims (2p, 2p + 1).
    """

    def __init__(self, sections, *, theta: float = 10000.0, frequencies: str = "axis", pairing: str = "halves"):
        sections = tuple(int(n) for n in sections)
        if not sections or any(n < 1 for n in sections):
            raise ValueError(f"sections must be positive numbers of pairs; got {sections}")
        if sum(sections) % 8 or sum(sections) > max(_DIMS) // 2:
            raise ValueError(f"sections must add up to a multiple of 8 of at most 128 pairs; got {sum(sections)}")
        if frequencies not in ("axis", "shared"):
            raise ValueError(f"frequencies must be 'axis' or 'shared' (got {frequencies!r})")
        if pairing not in ("halves", "adjacent"):
            raise ValueError(f"pairing must be 'halves' or 'adjacent' (got {pairing!r})")
        if not 0.0 < float(theta) < math.inf:
            raise ValueError(f"theta must be a positive finite number; got {theta}")
        self.sections = sections
        self.theta = float(theta)
        self.frequencies = frequencies
        self.pairing = pairing
        self._tables = {}  # device -> (turns for one position, axis) of each pair

    def _table(self, device):
        table = self._tables.get(device)
        if table is None:
            if torch.cuda.is_current_stream_capturing():
                raise RuntimeError(f"AxialRope: its table for {device} is made by the first call there, which a graph "
                                   "cannot capture: call it once before the capture")
            P = sum(self.sections)
            turns, axes = [], []
            for a, n in enumerate(self.sections):
                for i in range(n):
                    power = i / n if self.frequencies == "axis" else len(turns) / P
                    turns.append(self.theta ** -power / (2.0 * math.pi))
                    axes.append(a)
            table = self._tables[device] = (torch.tensor(turns, dtype=torch.float64, device=device),
                                            torch.tensor(axes, dtype=torch.int32, device=device))
        return table

    def __call__(self, q, k, positions, *, layout: str = "bhsd", inverse: bool = False, inplace: bool = False):
        """Rotates q and k (None: q alone) and returns both.

        q, k: bf16 [B, H, S, D] ("bhsd") or [B, S, H, D] ("bshd"), each with its own
        number of heads, any strides with a contiguous last dim and rows on 16-byte
        boundaries. positions: int32 [axes, S], the same for every batch row, or
        [axes, B, S]; any values and strides. ``inverse`` turns back: it undoes the
        rotation, and takes the gradient of the outputs to that of q and k (the op
        itself records no autograd graph). ``inplace`` writes q and k; otherwise the
        results are new contiguous tensors.
        """
        table = self._tables.get(q.device) if isinstance(q, torch.Tensor) else None
        if table is not None:
            res = _lib.calls.rope(q, k, positions, table[0], table[1], len(self.sections), layout,
                                  self.pairing == "halves", inverse, inplace)
            if res is not None:
                return res
        who = "AxialRope"
        if layout not in ("bhsd", "bshd"):
            raise ValueError(f"layout must be 'bhsd' or 'bshd' (got {layout!r})")
        sax, hax = (1, 2) if layout == "bshd" else (2, 1)
        P, A = sum(self.sections), len(self.sections)
        for name, t in (("q", q), ("k", k)):
            if name == "k" and t is None:
                continue
            ck.tensor(t, name, who, torch.bfloat16)
            if t.dim() != 4:
                raise ValueError(f"{who}: {name} must be 4-D ({layout.upper()}); got shape={tuple(t.shape)}")
            if t.shape[3] not in _DIMS or t.shape[3] != q.shape[3] or t.shape[3] < 2 * P:
                raise ValueError(f"{who}: head_dim must be 64, 128 or 256, the same for q and k, and at least {2 * P}; "
                                 f"got {name} of {t.shape[3]}")
            if t.shape[0] != q.shape[0] or t.shape[sax] != q.shape[sax] or t.shape[hax] < 1:
                raise ValueError(f"{who}: k must have q's batch and sequence, and both at least one head; "
                                 f"got {name} of shape {list(t.shape)}")
            ck.rows(t, name, who)
            if inplace:
                ck.one_place_each(t, name, who)
        if inplace and k is not None and not ck.share_none(q, k):
            raise ValueError(f"{who}: q and k must not share elements when they are written in place")
        B, S = q.shape[0], q.shape[sax]
        if not isinstance(positions, torch.Tensor) or positions.dtype != torch.int32:
            raise ValueError(f"{who}: positions must be int32")
        if tuple(positions.shape) not in ((A, S), (A, B, S)):
            raise ValueError(f"{who}: positions must be [{A}, {S}] or [{A}, {B}, {S}], got {list(positions.shape)}")
        dev = q.device
        ck.on_device(who, dev, k=k, positions=positions)
        pos = positions if positions.dim() == 3 else positions.unsqueeze(1).expand(A, B, S)
        with torch.cuda.device(dev):
            turns, axes = self._table(dev)
            outs = [t if inplace or t is None else torch.empty(t.shape, dtype=t.dtype, device=dev) for t in (q, k)]
            st = [t.stride(i) if t is not None else 0 for t in (q, k, *outs) for i in (0, sax, hax)]
            strides = (ctypes.c_longlong * 15)(*st, *pos.stride())
            p = _lib.ptr
            rc = _lib.lib.launch_rope_axes(p(q), p(k), p(outs[0]), p(outs[1]), p(pos), p(turns), p(axes), B, S,
                                           q.shape[hax], 0 if k is None else k.shape[hax], q.shape[3], P, A,
                                           int(self.pairing == "halves"), int(bool(inverse)), strides,
                                           _lib.stream_ptr(dev))
            if rc != 0:
                raise RuntimeError(f"launch_rope_axes returned error code {rc}")
        return outs[0], outs[1]
