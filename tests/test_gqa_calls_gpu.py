"""The native path (csrc/calls.cpp) of the paged-cache ops and AxialRope: it takes plain
GPU calls, gives what the Python path gives, and leaves what that refuses to it."""
import pytest
import torch

import moonmath_attention as ma
from gqa_inputs import cache, tables
from moonmath_attention import _lib

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


class _Off:
    def __getattr__(self, name):
        return lambda *a: None


def calls(fp8, order):
    k, v, ks, vs = cache(12, 2, 32, 64, fp8, 1, order)
    move = lambda t: None if t is None else t.to(DEV)  # noqa: E731
    k, v = (t.transpose(1, 2).contiguous().to(DEV).transpose(1, 2) if order == "tokens" else t.to(DEV) for t in (k, v))
    ks, vs = move(ks), move(vs)
    table = tables([200, 3], 32, 12, 1).to(DEV)
    n = torch.tensor([200, 3], dtype=torch.int32, device=DEV)
    g = torch.Generator(device=DEV).manual_seed(2)
    fused = torch.randn(2, 3, 10, 64, generator=g, device=DEV).bfloat16()
    slots = torch.tensor([5, 77, -1, 40, 41, 300], dtype=torch.int32, device=DEV)
    rows = fused.view(6, 10, 64)
    pos = torch.arange(6, dtype=torch.int32, device=DEV).view(2, 3)
    rope = ma.AxialRope((16, 16))
    rope(fused[:, :, :6], None, pos, layout="bshd")  # its table
    out = torch.empty(2, 3, 6, 64, dtype=torch.bfloat16, device=DEV)
    kk, vv = (torch.empty(6, 2, 64, dtype=torch.bfloat16, device=DEV) for _ in range(2))

    def run():
        got = [ma.gqa_decode_paged(fused[:, :, :6], k, v, n, table, k_scale=ks, v_scale=vs)]
        got += ma.gqa_decode_paged(fused[:, 0, :6], k, v, n, table, scale=0.3, k_scale=ks, v_scale=vs, return_lse=True)
        got.append(ma.gqa_decode_paged(fused[:, :, :6], k, v, n, table, k_scale=ks, v_scale=vs, out=out).clone())
        ma.gqa_kv_write(rows[:, 6:8], rows[:, 8:], k, v, slots, ks, vs)
        got += [t.clone() for t in (k, v, ks, vs) if t is not None]
        got += ma.gqa_kv_read(k, v, slots, ks, vs)
        got += [t.clone() for t in ma.gqa_kv_read(k, v, slots, ks, vs, k=kk, v=vv)]
        got += rope(fused[:, :, :6], fused[:, :, 6:8], pos, layout="bshd")
        got += rope(fused, fused[:, :, :3], pos.unsqueeze(1).expand(2, 3, 3)[..., 2].contiguous().unsqueeze(1)
                    .expand(2, 2, 3), layout="bshd", inverse=True)
        got.append(rope(fused.transpose(1, 2), None, pos, layout="bhsd")[0])
        return got

    return run


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("order", ["heads", "tokens"])
def test_native_equals_python(fp8, order, monkeypatch):
    run = calls(fp8, order)
    run()
    got = run()
    with monkeypatch.context() as m:
        m.setattr(_lib, "calls", _Off())
        want = run()
    torch.cuda.synchronize()
    for a, b in zip(got, want, strict=True):
        assert a.shape == b.shape and a.stride() == b.stride() and a.dtype == b.dtype
        assert torch.equal(a.contiguous().view(torch.uint8), b.contiguous().view(torch.uint8))


def test_plain_calls_are_taken():
    c = _lib.calls
    k, v, ks, vs = (t.to(DEV) for t in cache(4, 2, 16, 64, True, 3))
    q = torch.zeros(1, 4, 64, dtype=torch.bfloat16, device=DEV)
    n = torch.ones(1, dtype=torch.int32, device=DEV)
    t = torch.zeros(1, 2, dtype=torch.int32, device=DEV)
    x = torch.zeros(1, 2, 64, dtype=torch.bfloat16, device=DEV)
    turns, axes = ma.AxialRope((32,))._table(torch.device(DEV))
    p = torch.zeros(1, 4, dtype=torch.int32, device=DEV)
    r = torch.zeros(1, 4, 2, 64, dtype=torch.bfloat16, device=DEV)
    assert c.gqa_decode(q, k, v, n, t, None, ks, vs, None, False) is not None
    assert c.gqa_write(x, x, k, v, n, ks, vs) is True
    assert c.gqa_read(k, v, n, ks, vs, None, None) is not None
    assert c.rope(r, r, p, turns, axes, 1, "bshd", True, False, False) is not None
    # what the wrappers refuse, or handle themselves
    assert c.gqa_decode(q, k, v, n, t, None, ks, None, None, False) is None
    assert c.gqa_decode(q, k, v, n, t, None, ks, vs, q[:, :2], False) is None
    assert c.gqa_decode(q.requires_grad_(), k, v, n, t, None, ks, vs, None, False) is None
    assert c.gqa_write(x, x, k, k[:1].expand(4, 2, 16, 64), n, ks, vs) is None
    assert c.gqa_write(x, x[..., :32], k, v, n, ks, vs) is None
    assert c.gqa_read(k, v, n.long(), ks, vs, None, None) is None
    assert c.rope(r, r, p, turns, axes, 1, "bshd", True, False, True) is None
    assert c.rope(r, r, p.t(), turns, axes, 1, "bshd", True, False, False) is None
    torch.cuda.synchronize()


def test_caches_in_one_tensor_are_taken():
    c = _lib.calls
    n = torch.ones(1, dtype=torch.int32, device=DEV)
    x = torch.ones(1, 2, 64, dtype=torch.bfloat16, device=DEV)
    one = torch.zeros(4, 2, 2, 16, 64, dtype=torch.bfloat16, device=DEV)
    pairs = [(one[:, 0], one[:, 1]), (one[:, :, 1], one[:, :, 0]), (one.view(2, 4, 2, 16, 64)[0], one.view(2, 4, 2, 16, 64)[1]),
             tuple(one.view(4, 16, 2, 2, 64).select(3, i).transpose(1, 2) for i in (0, 1)),
             tuple(one.view(4, 2, 16, 128)[..., 64 * i:64 * i + 64] for i in (0, 1))]
    for k, v in pairs:
        one.zero_()
        assert c.gqa_write(x, 2 * x, k, v, n, None, None) is True
        assert k.float().sum() == 128 and v.float().sum() == 256
        assert c.gqa_write(x, x, k, k, n, None, None) is None
        assert c.gqa_write(x, x, k[1:], k[:-1], n, None, None) is None
    k, v = pairs[0]
    out = torch.empty(1, 2, 2, 64, dtype=torch.bfloat16, device=DEV)
    assert c.gqa_read(k, v, n, None, None, out[:, 0], out[:, 1]) is not None
    assert c.gqa_read(k, v, n, None, None, out[:, 0], out[:, 0]) is None
    torch.cuda.synchronize()


def test_refusals_on_the_gpu():
    k, v, _, _ = (None if t is None else t.to(DEV) for t in cache(4, 2, 16, 64, False, 3))
    q = torch.zeros(1, 4, 64, dtype=torch.bfloat16, device=DEV)
    n = torch.ones(1, dtype=torch.int32, device=DEV)
    t = torch.zeros(1, 2, dtype=torch.int32, device=DEV)
    for bad in ({"q": q.cpu()}, {"k": k.cpu()}, {"n": n.cpu()}, {"t": t.cpu()}):
        a = {"q": q, "k": k, "n": n, "t": t, **bad}
        with pytest.raises(ValueError, match="must be on"):
            ma.gqa_decode_paged(a["q"], a["k"], v, a["n"], a["t"])
    with pytest.raises(ValueError, match="apart"):
        ma.gqa_kv_write(k.view(-1, 2, 64)[:1], q[:, :2], k, v, n)
    with pytest.raises(ValueError, match="must be on"):
        ma.gqa_kv_read(k, v, n.cpu())
    with pytest.raises(ValueError, match="must be on"):
        ma.AxialRope((32,))(q[None], None, torch.zeros(1, 4, dtype=torch.int32))
