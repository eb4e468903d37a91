"""GPU tests of ``gqa_kv_write`` and ``gqa_kv_read``: bytes and scales equal to the
oracle's (oracle/gqa.py), rows of no token untouched; and a serving step with rotation,
writing, decoding and reading back together."""
import math

import pytest
import torch

import moonmath_attention as ma
from gqa_inputs import cache
from oracle import gqa as og

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.fixture(scope="module", autouse=True)
def _need_gpu():
    assert torch.cuda.is_available(), "GPU tests need an MI355X"


def empty_cache(nb, heads, page, D, fp8, order="heads", fill=0x5A):
    shape = (nb, heads, page, D) if order == "heads" else (nb, page, heads, D)
    made = []
    for _ in range(2):
        t = torch.full(shape + (() if fp8 else (2,)), fill, dtype=torch.uint8, device=DEV)
        t = t.view(torch.float8_e4m3fn) if fp8 else t.view(torch.bfloat16)[..., 0]
        t = t if fp8 else t.contiguous()
        made.append(t if order == "heads" else t.transpose(1, 2))
    scales = [torch.full((nb, heads, page), 7.5, device=DEV) if fp8 else None for _ in range(2)]
    return made + scales


def by_slot(t):
    """[nb, heads, page, ...] -> bytes (or values) by slot, on the CPU."""
    t = t.cpu()
    t = t.view(torch.uint8) if t.dtype == torch.float8_e4m3fn else t.view(torch.int16) if t.dtype == torch.bfloat16 else t
    return t.transpose(1, 2).reshape(t.shape[0] * t.shape[2], t.shape[1], *t.shape[3:])


def same_codes(a, b):
    """Equal e4m3fn bytes; of a NaN the sign does not count."""
    nan = (b & 0x7F) == 0x7F
    return torch.equal((a & 0x7F) == 0x7F, nan) and torch.equal(a[~nan], b[~nan])


def check_write(k, v, slots, c, before):
    nb, heads, page, D = c[0].shape
    live = (slots >= 0) & (slots < nb * page)
    at = slots[live].long()
    others = torch.ones(nb * page, dtype=torch.bool)
    others[at] = False
    for x, t, s, t0, s0 in zip((k, v), c[:2], c[2:], before[:2], before[2:]):
        got = by_slot(t)
        assert torch.equal(got[others], by_slot(t0)[others])
        if s is None:
            assert torch.equal(got[at], x[live].contiguous().view(torch.int16))
            continue
        codes, scale = og.quantize(x[live])
        assert torch.equal(by_slot(s)[at], scale)
        assert torch.equal(by_slot(s)[others], by_slot(s0)[others])
        assert same_codes(got[at], codes.view(torch.uint8))


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("N,heads,page,order", [(1, 1, 16, "heads"), (77, 3, 32, "tokens"), (1000, 8, 64, "heads"),
                                                (513, 2, 256, "tokens")])
def test_rows_match_oracle(N, heads, page, order, D, fp8):
    g = torch.Generator().manual_seed(N + D)
    nb = -(-N // page) + 3
    # rows of very different size: the smallest and largest scales, and rows of zeros
    size = torch.exp2(torch.randint(-120, 120, (N, heads, 1), generator=g).float())
    k, v = ((torch.randn(N, heads, D, generator=g) * size).to(torch.bfloat16) for _ in range(2))
    k[::13], v[::17] = 0.0, -0.0
    slots = torch.randperm(nb * page, generator=g)[:N].to(torch.int32)
    slots[5::31] = -1
    slots[6::31] = nb * page
    slots[7::31] = -2 ** 31
    slots[8::31] = 2 ** 31 - 1
    c = empty_cache(nb, heads, page, D, fp8, order)
    before = [None if t is None else t.clone() for t in c]
    ma.gqa_kv_write(k.to(DEV), v.to(DEV), c[0], c[1], slots.to(DEV), c[2], c[3])
    torch.cuda.synchronize()
    check_write(k, v, slots, c, before)


def test_every_bf16_value():
    """All 65536 patterns, each beside 63 others of one binade and sign so that scales
    and codes of every size occur; NaN and infinities give NaN codes and no scale."""
    pat = torch.arange(65536, dtype=torch.int32).to(torch.int16).view(torch.bfloat16).view(-1, 1, 64)
    mixed = pat.flatten().view(64, -1).t().contiguous().view(-1, 1, 64)  # and rows over all binades
    for k, v in ((pat, mixed), (mixed, pat)):
        N = k.shape[0]
        c = empty_cache(N // 16, 1, 16, 64, True)
        before = [t.clone() for t in c]
        slots = torch.arange(N, dtype=torch.int32)
        ma.gqa_kv_write(k.to(DEV), v.to(DEV), c[0], c[1], slots.to(DEV), c[2], c[3])
        torch.cuda.synchronize()
        # Scales under 2^-118 leave remainders that fp32 cannot hold: there a code may be
        # a neighbour's where the quotient lies within an fp32 step of a border.
        for x, t, s in ((k, c[0], c[2]), (v, c[1], c[3])):
            codes, scale = og.quantize(x)
            assert torch.equal(by_slot(s), scale)
            got, want = by_slot(t), codes.view(torch.uint8)
            plain = (scale > 2.0 ** -118)[..., None].expand_as(got)
            assert same_codes(got[plain], want[plain])
            a, b = (y.view(torch.float8_e4m3fn).float() for y in (got, want))
            assert torch.equal(a.isnan(), b.isnan())
            fine = ~b.isnan()
            near = (x.float().double() / scale.double()[..., None])[fine]
            assert ((a.double()[fine] - near).abs() <= near.abs() * 2.0 ** -4 * (1 + 2.0 ** -20) + 2.0 ** -10 * (1 + 2.0 ** -20)).all()
        del before


@pytest.mark.parametrize("fp8", [False, True])
def test_ties_round_to_even(fp8):
    """amax = 7 * 2^e * j makes the scale short and quotients lie exactly between codes."""
    rows = []
    for j in range(1, 37):
        x = torch.zeros(64)
        x[0] = 7.0 * j
        x[1:] = j / 64.0 * (torch.arange(63) + 1) / 2
        rows.append(x.to(torch.bfloat16))
    k = torch.stack(rows)[:, None].contiguous()
    c = empty_cache(3, 1, 16, 64, fp8)
    before = [None if t is None else t.clone() for t in c]
    slots = torch.arange(36, dtype=torch.int32)
    ma.gqa_kv_write(k.to(DEV), k.neg().to(DEV), c[0], c[1], slots.to(DEV), c[2], c[3])
    torch.cuda.synchronize()
    check_write(k, k.neg(), slots, c, before)


@pytest.mark.parametrize("fp8", [False, True])
def test_strides_of_rows_and_caches(fp8):
    """K and V slices of a fused projection, caches and scales slices of one tensor."""
    g = torch.Generator().manual_seed(3)
    fused = torch.randn(50, 12, 64, generator=g).to(torch.bfloat16)
    k, v = fused[:, 6:9], fused[:, 9:]
    d = fused.to(DEV)
    raw = torch.full((5, 3, 2, 16, 64 if fp8 else 128), 0x11, dtype=torch.uint8, device=DEV)
    both = raw.view(torch.float8_e4m3fn) if fp8 else raw.view(torch.bfloat16)
    sc = torch.full((5, 2, 3, 16), 3.0, device=DEV) if fp8 else None
    c = [both[:, :, 0], both[:, :, 1], sc[:, 0] if fp8 else None, sc[:, 1] if fp8 else None]
    before = [None if t is None else t.clone() for t in c]
    slots = torch.randperm(80, generator=g)[:50].to(torch.int32)
    ma.gqa_kv_write(d[:, 6:9], d[:, 9:], c[0], c[1], slots.to(DEV), c[2], c[3])
    torch.cuda.synchronize()
    check_write(k, v, slots, c, before)
    # read back into slices of one tensor, the same slots twice
    out = torch.full((100, 3, 2, 64), 5.0, dtype=torch.bfloat16, device=DEV)
    twice = torch.cat([slots, slots]).to(DEV)
    got = ma.gqa_kv_read(c[0], c[1], twice, c[2], c[3], k=out[:, :, 0], v=out[:, :, 1])
    assert got[0].data_ptr() == out.data_ptr()
    want = ma.gqa_kv_read(c[0], c[1], twice, c[2], c[3])
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    assert torch.equal(want[0][:50], want[0][50:])


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("D,order,page", [(64, "tokens", 16), (128, "heads", 64), (256, "heads", 128)])
def test_read_matches_oracle(D, order, page, fp8):
    """Rows by slot, zeros for padding tokens and slots past the cache; NaN stays NaN."""
    k, v, ks, vs = cache(7, 3, page, D, fp8, 5, order)
    (k.view(torch.uint8) if fp8 else k)[2, 1, 3, 5] = 0x7F if fp8 else math.nan
    g = torch.Generator().manual_seed(6)
    slots = torch.randint(-3, 7 * page + 3, (400,), generator=g).to(torch.int32)
    slots[0], slots[1], slots[2] = -2 ** 31, 2 ** 31 - 1, 2 * page + 3
    move = lambda t: t.transpose(1, 2).contiguous().to(DEV).transpose(1, 2) if order == "tokens" else t.to(DEV)  # noqa: E731
    got = ma.gqa_kv_read(move(k), move(v), slots.to(DEV), ks.to(DEV) if fp8 else None, vs.to(DEV) if fp8 else None)
    torch.cuda.synchronize()
    live = (slots >= 0) & (slots < 7 * page)
    at = slots[live].long()
    for x, t, s in zip(got, (k, v), (ks, vs)):
        x = x.cpu()
        assert (x[~live] == 0).all()
        want = t.float().transpose(1, 2).reshape(7 * page, 3, D)[at]
        if fp8:
            want = want * s.transpose(1, 2).reshape(7 * page, 3)[at][..., None]
        want = want.to(torch.bfloat16)
        nan = want.isnan()
        assert torch.equal(x[live].isnan(), nan) and torch.equal(x[live][~nan], want[~nan])


def test_written_rows_read_back():
    """What an fp8 cache gives back is within half a code's step and the bf16 rounding of
    what was written: |x| 2^-4 for normal codes, 2^-10 scale below them, and 2^-8."""
    g = torch.Generator().manual_seed(8)
    k, v = (torch.randn(300, 4, 128, generator=g).to(torch.bfloat16) for _ in range(2))
    c = empty_cache(5, 4, 64, 128, True)
    slots = torch.randperm(320, generator=g)[:300].to(torch.int32).to(DEV)
    ma.gqa_kv_write(k.to(DEV), v.to(DEV), c[0], c[1], slots, c[2], c[3])
    for x, y in zip((k, v), ma.gqa_kv_read(c[0], c[1], slots, c[2], c[3])):
        x, y = x.double(), y.cpu().double()
        s = x.abs().amax(-1, keepdim=True) / 448
        assert ((x - y).abs() <= (x.abs() * 2.0 ** -4).clamp(min=0) + 2.0 ** -10 * s + 1.07 * 2.0 ** -8 * x.abs()).all()


def test_no_token():
    c = empty_cache(2, 2, 16, 64, True)
    z = torch.zeros(0, 2, 64, dtype=torch.bfloat16, device=DEV)
    s = torch.zeros(0, dtype=torch.int32, device=DEV)
    ma.gqa_kv_write(z, z, c[0], c[1], s, c[2], c[3])
    k, v = ma.gqa_kv_read(c[0], c[1], s, c[2], c[3])
    assert k.shape == v.shape == (0, 2, 64)


def test_offsets_past_32_bits():
    nb = 40000
    c = [torch.zeros(nb, 16, 64, 128, dtype=torch.float8_e4m3fn, device=DEV) for _ in range(2)]
    c += [torch.zeros(nb, 16, 64, device=DEV) for _ in range(2)]
    g = torch.Generator().manual_seed(12)
    k, v = (torch.randn(5, 16, 128, generator=g).to(torch.bfloat16) for _ in range(2))
    slots = torch.tensor([nb * 64 - 1, 0, 33000 * 64 + 5, 20000 * 64, 16384 * 64 - 1], dtype=torch.int32)
    ma.gqa_kv_write(k.to(DEV), v.to(DEV), c[0], c[1], slots.to(DEV), c[2], c[3])
    got = ma.gqa_kv_read(c[0], c[1], slots.to(DEV), c[2], c[3])
    for x, t, s, y in zip((k, v), c[:2], c[2:], got):
        codes, scale = og.quantize(x)
        blk, row = (slots // 64).long().to(DEV), (slots % 64).long().to(DEV)
        assert torch.equal(t.view(torch.uint8)[blk, :, row].cpu(), codes.view(torch.uint8))
        assert torch.equal(s[blk, :, row].cpu(), scale)
        assert torch.equal(y.cpu(), (codes.float() * scale[..., None]).to(torch.bfloat16))
        assert int((t.view(torch.uint8)[:100] != 0).sum()) == int((codes[1].view(torch.uint8) != 0).sum())


def test_graph_replays():
    """A captured write and read, replayed with rows and slots changed in place."""
    g = torch.Generator(device=DEV).manual_seed(13)
    k, v = (torch.randn(64, 2, 64, generator=g, device=DEV).bfloat16() for _ in range(2))
    slots = torch.randperm(160, generator=g, device=DEV)[:64].to(torch.int32)
    a, b = empty_cache(10, 2, 16, 64, True), empty_cache(10, 2, 16, 64, True)
    ma.gqa_kv_write(k, v, a[0], a[1], slots, a[2], a[3])
    ma.gqa_kv_write(k, v, b[0], b[1], slots, b[2], b[3])
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ma.gqa_kv_write(k, v, a[0], a[1], slots, a[2], a[3])
        got = ma.gqa_kv_read(a[0], a[1], slots, a[2], a[3])
    for i in range(4):
        k.normal_(generator=g)
        v.normal_(generator=g)
        slots.copy_(torch.randperm(160, generator=g, device=DEV)[:64])
        slots[i] = -1
        graph.replay()
        torch.cuda.synchronize()
        ma.gqa_kv_write(k, v, b[0], b[1], slots, b[2], b[3])
        want = ma.gqa_kv_read(b[0], b[1], slots, b[2], b[3])
        for x, y in zip([*got, *a], [*want, *b]):
            assert torch.equal(x.view(torch.uint8), y.view(torch.uint8))


@pytest.mark.parametrize("fp8", [False, True])
def test_a_serving_step(fp8):
    """A prompt and then single tokens of two requests: rotated by three axes, written,
    decoded; each output against attention in 64 bits over the rows that the cache holds,
    and the last one against ``forward`` over the rows read back."""
    H, D, page, prompt, steps = 4, 128, 32, [45, 130], 6
    rope = ma.AxialRope((16, 24, 24), frequencies="shared")
    g = torch.Generator().manual_seed(14)
    nb = 16
    c = empty_cache(nb, H, page, D, fp8, fill=0)
    for s in c[2:]:
        if s is not None:
            s.fill_(1.0)
    table = torch.randperm(nb, generator=g)[:12].view(2, 6).to(torch.int32)
    slot = lambda b, t: table[b].long()[t // page] * page + t % page  # noqa: E731

    def qkv(n):
        return [torch.randn(1, n, H, D, generator=g).to(torch.bfloat16).to(DEV) for _ in range(3)]

    for b, n in enumerate(prompt):
        _, k, v = qkv(n)
        t = torch.arange(n)
        pos = torch.stack([t // 12, t // 4 % 3, t % 4]).to(torch.int32).to(DEV)
        _, k = rope(k, k, pos, layout="bshd")
        ma.gqa_kv_write(k[0], v[0], c[0], c[1], slot(b, t).to(torch.int32).to(DEV), c[2], c[3])
    for i in range(steps):
        lens = [n + i + 1 for n in prompt]
        q, k, v = (x.view(2, 1, H, D) for x in qkv(2))
        pos = torch.tensor([[n - 1] for n in lens], dtype=torch.int32, device=DEV).expand(3, 2, 1)
        q, k = rope(q, k, pos, layout="bshd")
        slots = torch.stack([slot(b, torch.tensor(n - 1)) for b, n in enumerate(lens)]).to(torch.int32).to(DEV)
        ma.gqa_kv_write(k[:, 0], v[:, 0], c[0], c[1], slots, c[2], c[3])
        n = torch.tensor(lens, dtype=torch.int32, device=DEV)
        out = ma.gqa_decode_paged(q, c[0], c[1], n, table.to(DEV), k_scale=c[2], v_scale=c[3])
        cpu = [None if t is None else t.cpu() for t in c]
        want, _, bound, _ = og.decode(q.cpu(), cpu[0], cpu[1], lens, table, None, cpu[2], cpu[3])
        assert ((out.cpu().double() - want).abs() <= bound).all()
    for b, n in enumerate(lens):
        k, v = ma.gqa_kv_read(c[0], c[1], slot(b, torch.arange(n)).to(torch.int32).to(DEV), c[2], c[3])
        ref = ma.forward(q[b:b + 1], k[None], v[None], layout="bshd", round_mode="rtne")
        # forward rounds P to bf16 (half a step of each, and 2^-8 of the output once more),
        # and the rows read back are rounded once (fp8): K's by 2^-8 of sum |q k|.
        x, kk, vv = q[b, 0].cpu().double(), k.cpu().double(), v.cpu().double()
        s = torch.einsum("hd,nhd->hn", x, kk) * D ** -0.5
        mag = torch.einsum("hd,nhd->hn", x.abs(), kk.abs()).amax(-1) * D ** -0.5
        a = torch.einsum("hn,nhd->hd", s.softmax(-1), vv.abs())
        e = og.U8 * (1 + (1 + 2 * mag[:, None] if fp8 else 0)) * a + 2 * og.U8 * a
        assert ((out[b, 0].cpu().double() - ref[0, 0].cpu().double()).abs() <= e + bound[b, 0]).all()
