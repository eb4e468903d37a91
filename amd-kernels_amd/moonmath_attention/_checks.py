"""Argument checks shared by the ops over strided tensors (gqa.py, rope.py)."""
import torch


def tensor(t, name, who, dtype):
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{who}: {name} must be torch.Tensor; got {type(t).__name__}")
    if t.dtype != dtype:
        raise ValueError(f"{who}: {name} must be {str(dtype).removeprefix('torch.')}, got {t.dtype}")
    if t.requires_grad and torch.is_grad_enabled():
        raise ValueError(f"{who}: {name} requires grad, and the op has no backward pass: detach it")


def rows(t, name, who):
    """Rows of the last dim are contiguous, and every one lies on a 16-byte boundary
    (the kernels' loads and stores are 16 bytes wide)."""
    if t.stride(-1) != 1:
        raise ValueError(f"{who}: {name}'s last dim must be contiguous")
    es = t.element_size()
    if t.data_ptr() % 16 or any(s * es % 16 for s, n in zip(t.stride()[:-1], t.shape[:-1]) if n > 1):
        raise ValueError(f"{who}: {name}'s rows must lie on 16-byte boundaries")


def one_place_each(t, name, who):
    """No two elements share memory (a tensor that is written): each dim steps over
    all that the smaller steps span."""
    span = 1
    for s, n in sorted((s, n) for s, n in zip(t.stride(), t.shape) if n > 1):
        if s < span:
            raise ValueError(f"{who}: {name} is written, and its elements must not share memory")
        span = s * (n - 1) + span


def on_device(who, dev, **tensors):
    if dev.type != "cuda":
        raise ValueError(f"{who}: tensors must be on a CUDA/HIP device")
    for name, t in tensors.items():
        if t is not None and t.device != dev:
            raise ValueError(f"{who}: {name} must be on {dev}, got {t.device}")


def extent(t):
    """First and last + 1 byte of a tensor's memory."""
    if t.numel() == 0:
        return t.data_ptr(), t.data_ptr()
    last = sum(s * (n - 1) for s, n in zip(t.stride(), t.shape))
    return t.data_ptr(), t.data_ptr() + (last + 1) * t.element_size()


def apart(a, b):
    (a0, a1), (b0, b1) = extent(a), extent(b)
    return a1 <= b0 or b1 <= a0


def share_none(a, b):
    """Whether two tensors of one type that are both written, each with its elements
    apart, are seen to share none: they lie apart, or are slices of one tensor (the
    same steps in the dims that reach past the gap between them, and within those
    steps all of one before all of the other)."""
    if apart(a, b):
        return True
    lo, hi = (a, b) if a.data_ptr() < b.data_ptr() else (b, a)
    gap = (hi.data_ptr() - lo.data_ptr()) // lo.element_size()
    dims = [i for i in range(a.dim()) if lo.shape[i] > 1 or hi.shape[i] > 1]
    outer = [i for i in dims if lo.stride(i) >= gap]
    if any(lo.stride(i) != hi.stride(i) for i in dims) or any(lo.shape[i] != hi.shape[i] for i in outer):
        return False
    reach = [sum(t.stride(i) * (t.shape[i] - 1) for i in dims if i not in outer) + 1 for t in (lo, hi)]
    span = gap + reach[1]
    for s, n in sorted((lo.stride(i), lo.shape[i]) for i in outer):
        if s < span:
            return False
        span += s * (n - 1)
    return reach[0] <= gap
