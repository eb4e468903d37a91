"""GPU tests of ``AxialRope`` against rotations in 64 bits (oracle/gqa.py)."""
import pytest
import torch

import moonmath_attention as ma
from oracle import gqa as og

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.fixture(scope="module", autouse=True)
def _need_gpu():
    assert torch.cuda.is_available(), "GPU tests need an MI355X"


def inputs(B, S, Hq, Hk, D, axes, far, seed=1):
    g = torch.Generator().manual_seed(seed)
    q, k = (torch.randn(B, S, H, D, generator=g).to(torch.bfloat16) for H in (Hq, Hk))
    return q, k, torch.randint(-far, far, (axes, B, S), generator=g).to(torch.int32)


def check(got, x, pos, sections, frequencies, pairing, inverse=False, theta=10000.0):
    want, bound = og.rope_bound(x, pos, sections, theta, frequencies, pairing, inverse)
    assert ((got.cpu().double() - want).abs() <= bound).all()


@pytest.mark.parametrize("pairing", ["halves", "adjacent"])
@pytest.mark.parametrize("frequencies", ["axis", "shared"])
@pytest.mark.parametrize("D,sections", [(128, (8, 28, 28)), (128, (16, 24, 24)), (64, (32,)), (64, (1, 3, 4)),
                                        (128, (5, 11)), (256, (16, 56, 56)), (256, (22, 21, 21, 64)), (64, (8,))])
def test_against_64_bits(D, sections, frequencies, pairing):
    """Whole and partial rotations, one to four axes, sections that end inside a thread's
    pairs; positions on both sides of zero."""
    rope = ma.AxialRope(sections, frequencies=frequencies, pairing=pairing)
    q, k, pos = inputs(2, 37, 5, 2, D, len(sections), 5000)
    for inverse in (False, True):
        yq, yk = rope(*(t.to(DEV) for t in (q, k, pos)), layout="bshd", inverse=inverse)
        check(yq, q, pos, sections, frequencies, pairing, inverse)
        check(yk, k, pos, sections, frequencies, pairing, inverse)
    hq, hk = rope(q.transpose(1, 2).contiguous().to(DEV), k.transpose(1, 2).contiguous().to(DEV), pos.to(DEV),
                  layout="bhsd", inverse=True)
    assert hq.is_contiguous() and torch.equal(hq.transpose(1, 2), yq) and torch.equal(hk.transpose(1, 2), yk)


@pytest.mark.parametrize("far", [1 << 20, 1 << 31])
def test_far_positions(far):
    """Angles of any int32 position keep their place in the turn."""
    q, k, pos = inputs(1, 300, 2, 1, 64, 2, far, 2)
    pos[:, 0, 0], pos[:, 0, 1] = -2 ** 31, 2 ** 31 - 1
    rope = ma.AxialRope((16, 16), theta=500000.0, frequencies="shared")
    yq, yk = rope(*(t.to(DEV) for t in (q, k, pos)), layout="bshd")
    check(yq, q, pos, (16, 16), "shared", "halves", theta=500000.0)
    check(yk, k, pos, (16, 16), "shared", "halves", theta=500000.0)


@pytest.mark.parametrize("B,S,Hq,Hk", [(1, 1, 1, 1), (3, 1, 40, 8), (1, 5, 71, 1), (70, 1, 3, 3), (1, 4099, 2, 2)])
def test_sizes(B, S, Hq, Hk):
    """One token, odd numbers of tokens and heads, and heads shared out over workgroups."""
    q, k, pos = inputs(B, S, Hq, Hk, 128, 1, 4096, 3)
    yq, yk = ma.AxialRope((64,))(*(t.to(DEV) for t in (q, k, pos)), layout="bshd")
    check(yq, q, pos, (64,), "axis", "halves")
    check(yk, k, pos, (64,), "axis", "halves")


def test_no_keys_no_tokens():
    rope = ma.AxialRope((32,))
    q, _, pos = inputs(2, 9, 3, 1, 64, 1, 50)
    y, none = rope(q.to(DEV), None, pos.to(DEV), layout="bshd")
    assert none is None
    check(y, q, pos, (32,), "axis", "halves")
    z = torch.zeros(2, 0, 3, 64, dtype=torch.bfloat16, device=DEV)
    y, _ = rope(z, z, torch.zeros(1, 0, dtype=torch.int32, device=DEV), layout="bshd")
    assert y.shape == z.shape


def test_strides_positions_and_places():
    """Slices of a fused projection, shared and strided positions, and in place: all as
    contiguous tensors give it, and what lies beside them is left."""
    sections = (8, 12, 12)
    rope = ma.AxialRope(sections, pairing="adjacent")
    q, k, pos = inputs(2, 50, 6, 2, 128, 3, 900, 4)
    pos = pos[:, :1].expand(3, 2, 50)
    fused = torch.randn(2, 50, 10, 128).to(torch.bfloat16)
    fused[:, :, :6], fused[:, :, 6:8] = q, k
    d = fused.to(DEV)
    wq, wk = rope(q.to(DEV), k.to(DEV), pos.contiguous().to(DEV), layout="bshd")
    check(wq, q, pos, sections, "axis", "adjacent")
    yq, yk = rope(d[:, :, :6], d[:, :, 6:8], pos[:, 0].to(DEV), layout="bshd")
    assert torch.equal(yq, wq) and torch.equal(yk, wk) and torch.equal(d.cpu(), fused)
    by_token = pos[:, 0].t().contiguous().to(DEV).t()  # strides (1, 3)
    yq, yk = rope(d[:, :, :6], d[:, :, 6:8], by_token, layout="bshd", inplace=True)
    assert yq.data_ptr() == d.data_ptr() and torch.equal(yq, wq) and torch.equal(yk, wk)
    assert torch.equal(d[:, :, 8:].cpu(), fused[:, :, 8:])


def test_there_and_back():
    """The inverse undoes the rotation up to the two roundings: 2^-8 of each value, and of
    the pair's other one through the second turn."""
    q, k, pos = inputs(1, 200, 3, 3, 128, 3, 100000, 5)
    rope = ma.AxialRope((16, 24, 24))
    p = pos.to(DEV)
    back = rope(*rope(q.to(DEV), k.to(DEV), p, layout="bshd"), p, layout="bshd", inverse=True)
    for x, y in zip((q, k), back):
        x, y = x.double(), y.cpu().double()
        pair = (x[..., :64].square() + x[..., 64:].square()).sqrt().repeat(1, 1, 1, 2)
        assert ((x - y).abs() <= og.U8 * (2 ** 0.5 * pair * 1.01 + x.abs() * 1.01) + 1e-5 * pair).all()


def test_inverse_is_the_gradient():
    """For loss = sum(w y): the inverse rotation of w against autograd through the formula
    in 64 bits, and against differences of the formula along random directions."""
    sections = (16, 24, 24)
    q, k, pos = inputs(1, 40, 2, 1, 128, 3, 3000, 6)
    w, _, _ = inputs(1, 40, 2, 1, 128, 3, 3000, 7)
    rope = ma.AxialRope(sections, frequencies="shared", pairing="adjacent")
    grad, _ = rope(w.to(DEV), None, pos.to(DEV), layout="bshd", inverse=True)
    x = q.double().requires_grad_(True)
    P = 64
    a = torch.cat([pos[i].double()[..., None] * 10000.0 ** -((sum(sections[:i]) + torch.arange(n).double()) / P)
                   for i, n in enumerate(sections)], -1)[:, :, None]
    y = torch.stack([x[..., 0::2] * a.cos() - x[..., 1::2] * a.sin(), x[..., 0::2] * a.sin() + x[..., 1::2] * a.cos()], -1)
    (y.flatten(-2) * w.double()).sum().backward()
    _, bound = og.rope_bound(w, pos, sections, 10000.0, "shared", "adjacent", True)
    assert ((grad.cpu().double() - x.grad).abs() <= bound).all()
    args = (pos, sections, 10000.0, "shared", "adjacent")
    for seed in range(4):
        d = torch.randn(q.shape, generator=torch.Generator().manual_seed(seed)).double()
        loss = lambda h: (og.rope(q.double() + h * d, *args) * w.double()).sum()  # noqa: E731
        slope = (loss(1e-3) - loss(-1e-3)) / 2e-3
        assert (slope - (grad.cpu().double() * d).sum()).abs() <= (bound * d.abs()).sum() + 1e-6


def test_graph_replays():
    rope = ma.AxialRope((8, 28, 28))
    q, k, pos = (t.to(DEV) for t in inputs(1, 64, 4, 2, 128, 3, 5000, 8))
    rope(q, k, pos, layout="bshd")
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = rope(q, k, pos, layout="bshd")
    for i in range(4):
        q.normal_()
        k.normal_()
        pos.add_(i * 37)
        graph.replay()
        torch.cuda.synchronize()
        want = rope(q, k, pos, layout="bshd")
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_first_call_cannot_be_captured():
    """The table is copied from the host by the first call on a device."""
    rope = ma.AxialRope((32,))
    q, k, pos = (t.to(DEV) for t in inputs(1, 8, 1, 1, 64, 1, 50))
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="call it once before the capture"):
        with torch.cuda.graph(graph):
            rope(q, k, pos, layout="bshd")
    y, _ = rope(q, k, pos, layout="bshd")
    check(y, q.cpu(), pos.cpu(), (32,), "axis", "halves")


def test_before_forward():
    """Rotated queries and keys attend by differences of positions: moving all positions
    by the same steps leaves the attention as it was, up to the roundings of q and k."""
    B, S, H, D = 1, 256, 2, 128
    q, k, pos = inputs(B, S, H, H, D, 3, 60, 9)
    v = torch.randn(B, S, H, D).to(torch.bfloat16).to(DEV)
    rope = ma.AxialRope((8, 28, 28), pairing="adjacent")
    outs = []
    for move in (0, 1000):
        yq, yk = rope(q.to(DEV), k.to(DEV), (pos + move).to(DEV), layout="bshd")
        outs.append(ma.forward(yq, yk, v, layout="bshd", round_mode="rtne").cpu().double())
    # q and k are off by 2^-8 each: scores by 2 * 2^-8 sum |q k|, in both runs
    x, y = q.double().transpose(1, 2), k.double().transpose(1, 2)
    pairs = lambda t: (t[..., 0::2].square() + t[..., 1::2].square()).sqrt()  # noqa: E731
    mag = 2 * (pairs(x) @ pairs(y).transpose(2, 3)).amax() * D ** -0.5
    assert (outs[0] - outs[1]).abs().max() <= 2 * (2 * og.U8 * mag + 2 * og.U8) * 2 * v.cpu().double().abs().max()
