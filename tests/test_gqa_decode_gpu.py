"""GPU tests of ``gqa_decode_paged`` against the 64-bit oracle (oracle/gqa.py), whose
bound counts the kernel's roundings: half a step of bf16 for the output, fp32 sums,
and a P of two bf16 parts."""
import math

import pytest
import torch

import moonmath_attention as ma
from gqa_inputs import cache, poison, tables
from oracle import gqa as og

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
INF, NAN = math.inf, math.nan


@pytest.fixture(scope="module", autouse=True)
def _need_gpu():
    assert torch.cuda.is_available(), "GPU tests need an MI355X"


def gpu(*ts):
    return [None if t is None else t.to(DEV) for t in ts]


def keep_layout(t):
    """The same strides on the GPU."""
    if t is None:
        return None
    return t.to(DEV) if t.is_contiguous() else t.transpose(1, 2).contiguous().to(DEV).transpose(1, 2)


def rand_q(B, T, Hq, D, seed, peak=2.0):
    g = torch.Generator().manual_seed(seed + 9)
    return (torch.randn(B, T, Hq, D, generator=g) * peak).to(torch.bfloat16)


def check(got, lse, q, k, v, lens, table, scale=None, ks=None, vs=None):
    want, want_lse, bound, lse_bound = og.decode(q, k, v, lens, table, scale, ks, vs)
    got, lse = got.cpu().double(), lse.cpu().double()
    assert torch.equal(got.isnan(), want.isnan())
    assert torch.equal(got.isinf(), want.isinf()) and torch.equal(got[got.isinf()], want[want.isinf()])
    fine = want.isfinite()
    over = ((got - want).abs() - bound)[fine]
    assert over.numel() == 0 or over.max() <= 0, f"off by {((got - want).abs() / bound)[fine].max():.3g} bounds"
    assert torch.equal(lse.isnan(), want_lse.isnan())
    empty = want_lse == -INF
    assert torch.equal(lse == -INF, empty)
    fine = want_lse.isfinite()
    assert ((lse - want_lse).abs() <= lse_bound)[fine].all()


def run_case(lens, Hq, Hkv, D, T, page, fp8, order, seed=1, width=None):
    need = sum(-(-max(n, 0) // page) for n in lens)
    k, v, ks, vs = cache(need + 3, Hkv, page, D, fp8, seed, order)
    table = tables(lens, page, need + 3, seed, width)
    shown = [n if width is None else min(n, width * page) for n in lens]
    poison(k, v, ks, vs, table, shown)
    q = rand_q(len(lens), T, Hq, D, seed)
    n = torch.tensor(lens, dtype=torch.int32)
    out, lse = ma.gqa_decode_paged(q.to(DEV), keep_layout(k), keep_layout(v), n.to(DEV), table.to(DEV),
                                   k_scale=keep_layout(ks), v_scale=keep_layout(vs), return_lse=True)
    torch.cuda.synchronize()
    check(out, lse, q, k, v, lens, table, None, ks, vs)


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("Hq,Hkv", [(4, 4), (8, 2), (24, 1), (40, 1)])
def test_dims_and_groups(D, fp8, Hq, Hkv):
    """1, 4, 24 and 40 query rows for a kv head: one, two and four tiles of 16, in
    blocks; requests from no token to several tiles."""
    run_case([200, 1, 0, 129, 1000], Hq, Hkv, D, 1, 64, fp8, "heads", seed=D + Hq)


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("order", ["heads", "tokens"])
@pytest.mark.parametrize("page", [16, 32, 64, 128, 256, 1024])
def test_pages_and_orders(page, order, fp8):
    """Pages that end inside a step, a tile and beyond one."""
    run_case([1, 15, 16, 17, 31, 32, 33, 127, 128, 129, 255, 300, 700], 6, 3, 64, 1, page, fp8, order, seed=page)


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("T", [2, 3, 5, 8])
def test_draft_windows(T, fp8):
    """Windows at each place of a 32-token step and across two; requests shorter than
    the window leave its first queries without a token."""
    lens = [0, 1, 2, 3, 7, 8, 9, 31, 32, 33, 34, 37, 63, 64, 65, 66, 127, 128, 129, 133, 160, 256, 511, 513]
    run_case(lens, 8, 2, 128, T, 32, fp8, "heads", seed=T)


@pytest.mark.parametrize("D,Hq,Hkv,T", [(64, 16, 2, 8), (128, 48, 1, 8), (256, 16, 1, 4), (64, 71, 1, 3)])
def test_many_rows(D, Hq, Hkv, T):
    """64 to 384 query rows for a kv head, the last block of them partly filled; rows
    of one position in two blocks."""
    run_case([70, 5, 300, 1100], Hq, Hkv, D, T, 64, True, "tokens", seed=Hq)


# A table far wider than the requests makes a call be laid out as for long ones: rows of
# one kv head over several waves, neighbouring heads together, and always shared out.
WIDE = 4000  # pages of 16


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("Hq,Hkv,T,order", [
    (4, 2, 1, "heads"), (24, 1, 1, "heads"), (24, 1, 1, "tokens"), (16, 1, 2, "heads"), (48, 1, 1, "heads"),
    (33, 1, 3, "tokens"), (48, 1, 8, "heads"), (8, 2, 3, "tokens"), (8, 4, 2, "tokens"), (12, 6, 1, "tokens"),
    (40, 2, 2, "tokens")])
def test_layouts_of_long_calls(D, fp8, Hq, Hkv, T, order):
    """1 to 384 query rows for a kv head, one to eight kv heads."""
    lens = [0, 1, 2, 31, 33, 64, 65, 100, 129, 255, 300, 513, 640, 1000]
    run_case(lens, Hq, Hkv, D, T, 16, fp8, order, seed=Hq + T, width=WIDE)


@pytest.mark.parametrize("T", [1, 2, 5, 8])
@pytest.mark.parametrize("Hq,Hkv", [(8, 4), (64, 4), (17, 1)])
def test_windows_in_long_calls(T, Hq, Hkv):
    """Ends of requests at each place of two steps, where one group of waves has all steps
    and where several share them."""
    run_case([1, 2, 7, 8, 9] + list(range(28, 42)) + [63, 64, 65, 70, 96, 97], Hq, Hkv, 64, T, 16, False, "tokens", seed=T,
             width=WIDE)


@pytest.mark.parametrize("D,B,width,fp8", [(64, 100, 60, False), (64, 100, 60, True), (128, 150, 32, False),
                                           (128, 150, 32, True)])
def test_many_short_requests_of_many_rows(D, B, width, fp8):
    """24 rows for each workgroup that takes a request whole."""
    run_case([(37 * i) % (16 * width - 1) if i % 9 == 0 else i % 50 for i in range(B)], 24, 1, D, 1, 16, fp8, "heads", seed=B,
             width=width)


def test_a_large_batch():
    """More requests than threads look for a run's first one; most of them empty in places."""
    run_case([(7 * i) % 70 if i % 600 > 40 or i % 7 == 0 else 0 for i in range(1500)], 2, 2, 64, 2, 16, False, "heads",
             width=200)


@pytest.mark.parametrize("bad", [NAN, INF, -INF])
@pytest.mark.parametrize("Hq,Hkv,width", [(48, 1, WIDE), (8, 4, WIDE), (64, 2, 60), (4, 4, 20)])
def test_hidden_values_in_every_layout(bad, Hq, Hkv, width):
    """V of the last three drafts is not finite: each query takes those it sees."""
    lens = [300, 33, 34, 64]
    k, v, _, _ = cache(40, Hkv, 16, 64, False, 16, "tokens")
    table = tables(lens, 16, 40, 16, width)
    for b, n in enumerate(lens):
        for t in range(n - 3, n):
            v[table[b, t // 16], :, t % 16, 5 + t % 3] = bad
    q = rand_q(4, 4, Hq, 64, 16)
    out, lse = ma.gqa_decode_paged(q.to(DEV), keep_layout(k), keep_layout(v), torch.tensor(lens, dtype=torch.int32).to(DEV),
                                   table.to(DEV), return_lse=True)
    check(out, lse, q, k, v, lens, table)


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("lens", [[4097], [20000, 3], [65537], [0, 0, 0], [1] * 600, [0] * 299 + [513], [513, 0] * 150])
def test_lengths(lens, fp8):
    """One long request over all workgroups, uneven ones, many, and empty ones among
    them (more than the 256 that are planned at once)."""
    run_case(lens, 4, 2 if len(lens) > 9 else 1, 64, 1, 64, fp8, "heads", seed=len(lens))


def test_lengths_are_clamped():
    """Negative lengths are empty, lengths past the table end with it."""
    run_case([-5, 1000, 300, -2 ** 31, 2 ** 31 - 1][:3], 4, 2, 128, 2, 16, False, "heads", width=17)
    k, v, _, _ = cache(6, 2, 16, 128, False, 4)
    table = torch.tensor([[0, 1, 2], [3, 4, 5]], dtype=torch.int32)
    q = rand_q(2, 1, 4, 128, 4)
    out, lse = ma.gqa_decode_paged(*gpu(q, k, v), torch.tensor([2 ** 31 - 1, -2 ** 31], dtype=torch.int32).to(DEV),
                                   table.to(DEV), return_lse=True)
    check(out, lse, q, k, v, [48, 0], table)


def test_page_ids_are_clamped():
    """Ids outside the cache read its first or last block (the oracle clamps too)."""
    k, v, _, _ = cache(4, 1, 16, 64, False, 5)
    table = torch.tensor([[-1, 2 ** 31 - 1, 1, -2 ** 31, 4, 0, 3, 2, 1, 100]], dtype=torch.int32)
    q = rand_q(1, 1, 2, 64, 5)
    out, lse = ma.gqa_decode_paged(*gpu(q, k, v), torch.tensor([155], dtype=torch.int32).to(DEV), table.to(DEV),
                                   return_lse=True)
    check(out, lse, q, k, v, [155], table)


@pytest.mark.parametrize("T", [1, 4])
@pytest.mark.parametrize("at", [0, 40, 599])
@pytest.mark.parametrize("bad", [NAN, INF, -INF])
@pytest.mark.parametrize("which", ["k", "v"])
def test_values_that_are_not_finite(which, bad, at, T):
    """A NaN or infinity in a row of K or V reaches the queries that see the token, as
    the formula says, and no other: token 599 of 600 is seen by the last query only."""
    k, v, _, _ = cache(12, 2, 64, 128, False, 6)
    table = tables([600, 90], 64, 12, 6)
    (k if which == "k" else v)[table[0, at // 64], 0, at % 64, 5] = bad
    q = rand_q(2, T, 4, 128, 6)
    q[..., 5] = 1.5  # the score takes the infinity's sign
    out, lse = ma.gqa_decode_paged(*gpu(q, k, v), torch.tensor([600, 90], dtype=torch.int32).to(DEV), table.to(DEV),
                                   return_lse=True)
    if which == "k" and bad == INF:
        seen = torch.arange(T) + 600 - T + 1 > at  # inf - inf: NaN in every dim
        assert out[0, :, :2].isnan().cpu().eq(seen[:, None, None]).all() and not out[0, :, 2:].isnan().any()
        assert not out[1].isnan().any()
        return
    check(out, lse, q, k, v, [600, 90], table)


@pytest.mark.parametrize("lens,lost", [([600], 300), ([600], 600), ([5000], 4200), ([5000], 5000), ([40], 40)])
def test_scores_of_minus_infinity(lens, lost):
    """Tokens whose scores are -inf weigh nothing, also where they fill whole steps and
    runs; where all are, the softmax is 0 / 0 and its sum's ln is -inf."""
    n = -(-lens[0] // 64)
    k, v, _, _ = cache(n, 1, 64, 64, False, 7)
    table = tables(lens, 64, n, 7)
    t = torch.arange(lost)
    k[table[0].long()[t // 64], 0, t % 64, 3] = -INF
    q = rand_q(1, 1, 3, 64, 7)
    q[..., 3] = 0.5
    out, lse = ma.gqa_decode_paged(*gpu(q, k, v), torch.tensor(lens, dtype=torch.int32).to(DEV), table.to(DEV),
                                   return_lse=True)
    if lost == lens[0]:
        assert out.isnan().all() and (lse == -INF).all()
    else:
        check(out, lse, q, k, v, lens, table)


def test_large_and_small_scores():
    """Scores of thousands (one token takes all), a scale of its own, and a negative one."""
    k, v, _, _ = cache(20, 2, 64, 128, False, 8)
    table = tables([1200], 64, 20, 8)
    n = torch.tensor([1200], dtype=torch.int32)
    for peak, scale in ((100.0, None), (1.0, 3.0), (1.0, -0.2), (1.0, 0.0)):
        q = rand_q(1, 2, 4, 128, 8, peak)
        out, lse = ma.gqa_decode_paged(*gpu(q, k, v, n, table), scale=scale, return_lse=True)
        check(out, lse, q, k, v, [1200], table, scale)


@pytest.mark.parametrize("fp8", [False, True])
def test_strides(fp8):
    """q of a fused projection, K and V (and scales) slices of one tensor, a table that
    is part of a wider one, out of other strides: what contiguous tensors give."""
    lens = [300, 77, 1]
    k, v, ks, vs = cache(10, 2, 64, 64, fp8, 9)
    table = tables(lens, 64, 10, 9)
    q = rand_q(3, 3, 6, 64, 9)
    n = torch.tensor(lens, dtype=torch.int32).to(DEV)
    want = ma.gqa_decode_paged(*gpu(q, k, v), n, table.to(DEV), k_scale=gpu(ks)[0], v_scale=gpu(vs)[0])
    both = torch.stack([k.view(torch.uint8) if fp8 else k, v.view(torch.uint8) if fp8 else v], 2).to(DEV)
    k2, v2 = both[:, :, 0], both[:, :, 1]
    if fp8:
        k2, v2 = k2.view(torch.float8_e4m3fn), v2.view(torch.float8_e4m3fn)
        sc = torch.stack([ks, vs], 1).to(DEV)
        ks, vs = sc[:, 0], sc[:, 1]
    fused = torch.randn(3, 3, 10, 64, device=DEV).bfloat16()
    fused[:, :, :6] = q.to(DEV)
    wide = torch.full((3, 40), -1, dtype=torch.int32, device=DEV)
    wide[:, 4:4 + table.shape[1]] = table.to(DEV)
    out = torch.full((3, 6, 3, 64), 7.0, dtype=torch.bfloat16, device=DEV).transpose(1, 2)
    got = ma.gqa_decode_paged(fused[:, :, :6], k2, v2, n, wide[:, 4:4 + table.shape[1]], k_scale=ks, v_scale=vs, out=out)
    assert got is out and torch.equal(got, want)
    # in q's own place, and one query as a 3-D tensor
    mine = q.to(DEV).clone()
    assert torch.equal(ma.gqa_decode_paged(mine, k2, v2, n, table.to(DEV), k_scale=ks, v_scale=vs, out=mine), want)
    one, l1 = ma.gqa_decode_paged(q[:, 2].to(DEV), k2, v2, n, table.to(DEV), k_scale=ks, v_scale=vs, return_lse=True)
    four, l4 = ma.gqa_decode_paged(q[:, 2:].to(DEV), k2, v2, n, table.to(DEV), k_scale=ks, v_scale=vs, return_lse=True)
    assert one.shape == (3, 6, 64) and l1.shape == (3, 6) and torch.equal(one, four[:, 0]) and torch.equal(l1, l4[:, 0])


def test_offsets_past_32_bits():
    """Blocks of a cache of 9 GB, whose rows lie past 2^32 bytes and 2^31 elements."""
    nb = 36000
    k = torch.zeros(nb, 16, 64, 128, dtype=torch.bfloat16, device=DEV)
    v = torch.zeros_like(k)
    sk, sv, _, _ = cache(5, 16, 64, 128, False, 10)
    ids = torch.tensor([nb - 1, 17000, 0, nb - 2, 33333])
    k[ids.to(DEV)], v[ids.to(DEV)] = sk.to(DEV), sv.to(DEV)
    table = torch.arange(5, dtype=torch.int32)[None]
    q = rand_q(1, 1, 32, 128, 10)
    n = torch.tensor([5 * 64 - 3], dtype=torch.int32).to(DEV)
    out, lse = ma.gqa_decode_paged(q.to(DEV), k, v, n, ids.to(torch.int32)[None].to(DEV), return_lse=True)
    check(out, lse, q, sk, sv, [5 * 64 - 3], table)


def test_no_request():
    k, v, _, _ = gpu(*cache(2, 2, 16, 64, False, 1))
    i = torch.zeros(0, dtype=torch.int32, device=DEV)
    out, lse = ma.gqa_decode_paged(torch.zeros(0, 3, 4, 64, dtype=torch.bfloat16, device=DEV), k, v, i,
                                   torch.zeros(0, 2, dtype=torch.int32, device=DEV), return_lse=True)
    assert out.shape == (0, 3, 4, 64) and lse.shape == (0, 3, 4)


def _serving(seed, fp8=True, B=24, T=2):
    g = torch.Generator().manual_seed(seed)
    lens = torch.randint(0, 3000, (B,), generator=g).tolist()
    nb = sum(-(-n // 64) for n in lens) + B
    k, v, ks, vs = cache(nb, 2, 64, 64, fp8, seed)
    table = tables(lens, 64, nb, seed, width=47).clamp_(0, nb - 1)
    return gpu(rand_q(B, T, 8, 64, seed), k, v, torch.tensor(lens, dtype=torch.int32), table, ks, vs)


def _call(s, **more):
    return ma.gqa_decode_paged(s[0], s[1], s[2], s[3], s[4], k_scale=s[5], v_scale=s[6], return_lse=True, **more)


def test_the_same_call_gives_the_same_bits():
    s = _serving(3)
    want = _call(s)
    for _ in range(3):
        got = _call(s)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_calls_on_two_streams():
    """Calls that overlap share no workspace."""
    a, b = _serving(4), _serving(5, B=40, T=1)
    want = _call(a), _call(b)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(6):
        for i, s in enumerate((a, b)):
            with torch.cuda.stream(streams[i]):
                got[i].append(_call(s))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(o, want[i][0]) and torch.equal(l, want[i][1]) for o, l in got[i])


def test_graph_replays():
    """Two captured graphs, replayed in turn with lengths, tables and queries changed in
    place and eager work between: each replay equals the eager call."""
    states = [_serving(6), _serving(7)]
    graphs, outs = [], []
    for s in states:
        _call(s)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(_call(s))
        graphs.append(g)
    for i in range(4):
        for s, g, o in zip(states, graphs, outs):
            other = _serving(20 + i)
            s[0].copy_(other[0])
            s[3].copy_((s[3] * 7 + 13 * i) % 3000)
            s[4].copy_(s[4].roll(i, 0))
            g.replay()
            torch.cuda.synchronize()
            want = _call(s)
            assert torch.equal(o[0], want[0]) and torch.equal(o[1], want[1])


def test_graphs_of_one_pool():
    """Graphs that take workspaces and outputs from one pool, replayed one behind the
    other: each finds what it needs, and the first one's output is read before the next."""
    states = [_serving(8), _serving(9, B=40, T=1)]
    want = [_call(s) for s in states]
    pool = torch.cuda.graph_pool_handle()
    graphs, outs = [], []
    for s in states:
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, pool=pool):
            outs.append(_call(s))
        graphs.append(g)
    for i in (0, 1, 1, 0, 0, 1):
        graphs[i].replay()
        o, l = (t.clone() for t in outs[i])
        assert torch.equal(o, want[i][0]) and torch.equal(l, want[i][1])


def test_calls_from_two_threads():
    import threading

    states = [_serving(10), _serving(11, B=40, T=1)]
    want = [_call(s) for s in states]
    torch.cuda.synchronize()
    wrong = []

    def run(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(20):
                got = _call(states[i])
                torch.cuda.current_stream().synchronize()
                if not all(torch.equal(x, y) for x, y in zip(got, want[i])):
                    wrong.append(i)

    threads = [threading.Thread(target=run, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


def test_parts_join_by_their_sums():
    """A context cut at a page: its parts' outputs joined by their lse equal the whole's."""
    k, v, _, _ = cache(32, 2, 64, 128, False, 11)
    table = tables([2000], 64, 32, 11)
    q = rand_q(1, 1, 8, 128, 11).to(DEV)
    kd, vd, td = gpu(k, v, table)
    n = lambda x: torch.tensor([x], dtype=torch.int32, device=DEV)  # noqa: E731
    o1, l1 = ma.gqa_decode_paged(q, kd, vd, n(1024), td, return_lse=True)
    o2, l2 = ma.gqa_decode_paged(q, kd, vd, n(2000 - 1024), td[:, 16:], return_lse=True)
    w = torch.softmax(torch.stack([l1, l2]).double(), 0)[..., None]
    joined = w[0] * o1.double() + w[1] * o2.double()
    want, _, bound, _ = og.decode(q.cpu(), k, v, [2000], table)
    # two roundings to bf16 of the parts, each weighted, on top of the bound
    slack = og.U8 * (w[0] * o1.double().abs() + w[1] * o2.double().abs()).cpu()
    assert ((joined.cpu() - want).abs() <= bound + slack).all()
