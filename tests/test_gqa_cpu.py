"""CPU tests of the paged K/V cache ops and AxialRope: what they refuse and how, the
launchers' argument codes, and the oracle (oracle/gqa.py) against library routines."""
import ctypes
import math

import pytest
import torch

import moonmath_attention as ma
from gqa_inputs import cache, tables
from moonmath_attention import _checks, _lib
from oracle import gqa as og

BF, FP8, I32 = torch.bfloat16, torch.float8_e4m3fn, torch.int32


def z(*shape, dtype=BF):
    return torch.zeros(*shape, dtype=dtype)


def good(fp8=False):
    k, v, ks, vs = cache(6, 2, 16, 64, fp8, 1)
    return {"k_cache": k, "v_cache": v, "k_scale": ks, "v_scale": vs}


def decode(**change):
    a = {"q": z(3, 4, 64), "seq_lens": z(3, dtype=I32), "block_table": z(3, 2, dtype=I32), **good(), **change}
    return ma.gqa_decode_paged(a.pop("q"), a.pop("k_cache"), a.pop("v_cache"), a.pop("seq_lens"), a.pop("block_table"), **a)


def write(**change):
    a = {"k": z(5, 2, 64), "v": z(5, 2, 64), "slots": z(5, dtype=I32), **good(), **change}
    return ma.gqa_kv_write(a["k"], a["v"], a["k_cache"], a["v_cache"], a["slots"], a["k_scale"], a["v_scale"])


def read(**change):
    a = {"slots": z(5, dtype=I32), "k": None, "v": None, **good(), **change}
    return ma.gqa_kv_read(a["k_cache"], a["v_cache"], a["slots"], a["k_scale"], a["v_scale"], k=a["k"], v=a["v"])


@pytest.mark.parametrize("call", [decode, write, read])
def test_good_arguments_reach_the_device_check(call):
    with pytest.raises(ValueError, match="must be on a CUDA/HIP device"):
        call()
    with pytest.raises(ValueError, match="must be on a CUDA/HIP device"):
        call(**good(True))


_K64 = z(6, 2, 16, 64)
BAD_CACHES = [
    ({"k_cache": None}, TypeError, "must be torch.Tensor"),
    ({"k_cache": _K64.float()}, ValueError, "bfloat16 or float8_e4m3fn"),
    ({"k_cache": z(6, 2, 64)}, ValueError, "num_blocks, Hkv, page, D"),
    ({"k_cache": z(6, 2, 16, 96)}, ValueError, "D 64, 128 or 256"),
    ({"v_cache": z(6, 2, 32, 64)}, ValueError, "must be k_cache's"),
    ({"v_cache": _K64.to(FP8)}, ValueError, "v_cache must be bfloat16"),
    ({"k_cache": z(0, 2, 16, 64), "v_cache": z(0, 2, 16, 64)}, ValueError, "at least one block"),
    ({"k_cache": z(6, 2, 8, 64), "v_cache": z(6, 2, 8, 64)}, ValueError, "power of two"),
    ({"k_cache": z(6, 2, 48, 64), "v_cache": z(6, 2, 48, 64)}, ValueError, "power of two"),
    ({"k_cache": z(6, 2, 16, 128)[..., ::2], "v_cache": _K64}, ValueError, "last dim must be contiguous"),
    ({"k_cache": z(6, 2, 16, 68)[..., :64], "v_cache": _K64}, ValueError, "16-byte boundaries"),
    ({"k_cache": z(6 * 2 * 16 * 64 + 4)[4:].view(6, 2, 16, 64)}, ValueError, "16-byte boundaries"),
    ({"k_scale": z(6, 2, 16, dtype=torch.float32)}, ValueError, "go with a float8_e4m3fn cache"),
    ({**good(True), "v_scale": None}, ValueError, "go with a float8_e4m3fn cache"),
    ({**good(True), "k_scale": z(6, 2, 16)}, ValueError, "k_scale must be float32"),
    ({**good(True), "k_scale": z(6, 16, 2, dtype=torch.float32)}, ValueError, "num_blocks, Hkv, page"),
    ({**good(True), "k_scale": z(6, 16, 2, dtype=torch.float32).transpose(1, 2)}, ValueError, "must be contiguous"),
    ({**good(True), "k_scale": z(6, 2, 18, dtype=torch.float32)[..., :16]}, ValueError, "16-byte boundaries"),
    ({"k_cache": z(6, 2, 16, 64).requires_grad_()}, ValueError, "requires grad"),
]


@pytest.mark.parametrize("call", [decode, write, read])
@pytest.mark.parametrize("change,error,match", BAD_CACHES)
def test_refused_caches(call, change, error, match):
    with pytest.raises(error, match=match):
        call(**change)


def test_refused_distance_of_tokens():
    """A lane adds 15 rows in 32 bits. (The storage is never touched.)"""
    far = torch.empty(15 * ((1 << 26) + 8) + 64, dtype=BF).as_strided((1, 1, 16, 64), (0, 0, (1 << 26) + 8, 1))
    with pytest.raises(ValueError, match="2\\^26"):
        read(k_cache=far, v_cache=z(1, 1, 16, 64))


@pytest.mark.parametrize("change,error,match", [
    ({"q": None}, TypeError, "q must be torch.Tensor"),
    ({"q": z(3, 4, 64, dtype=torch.float16)}, ValueError, "q must be bfloat16"),
    ({"q": z(3, 64)}, ValueError, "q must be \\[B, Hq"),
    ({"q": z(3, 4, 128)}, ValueError, "q must be \\[B, Hq, 64\\]"),
    ({"q": z(3, 9, 4, 64)}, ValueError, "q_len must be in \\[1,8\\]"),
    ({"q": z(3, 0, 4, 64)}, ValueError, "q_len must be in \\[1,8\\]"),
    ({"q": z(3, 3, 64)}, ValueError, "multiple of the cache's 2 heads"),
    ({"q": z(3, 0, 64)}, ValueError, "multiple of the cache's 2 heads"),
    ({"q": z(3, 4, 68)[..., :64]}, ValueError, "16-byte boundaries"),
    ({"q": z(3, 4, 128)[..., ::2]}, ValueError, "last dim must be contiguous"),
    ({"q": z(3, 4, 64).requires_grad_()}, ValueError, "requires grad"),
    ({"seq_lens": z(3, dtype=torch.int64)}, ValueError, "seq_lens must be int32"),
    ({"seq_lens": z(4, dtype=I32)}, ValueError, "seq_lens must be contiguous \\[B\\]"),
    ({"seq_lens": z(6, dtype=I32)[::2]}, ValueError, "seq_lens must be contiguous \\[B\\]"),
    ({"block_table": [[0, 1]]}, ValueError, "block_table must be int32"),
    ({"block_table": z(2, 2, dtype=I32)}, ValueError, "block_table must be \\[B, max_blocks\\]"),
    ({"block_table": z(3, 0, dtype=I32)}, ValueError, "block_table must be \\[B, max_blocks\\]"),
    ({"block_table": z(2, 3, dtype=I32).t()}, ValueError, "last dim must be contiguous"),
    ({"block_table": z(3, 1, dtype=I32).expand(3, 1 << 27)}, ValueError, "at most 2\\^31 - 4096 tokens"),
    ({"q": z(1, 1, 64).expand(3, 65538, 64)}, ValueError, "at most 65536"),
    ({"scale": "x"}, ValueError, "could not convert"),
    ({"out": z(3, 4, 64, dtype=torch.float32)}, ValueError, "out must be bfloat16"),
    ({"out": z(3, 1, 4, 64)}, ValueError, "out must have q's shape"),
    ({"out": z(3, 1, 64).expand(3, 4, 64)}, ValueError, "must not share memory"),
    ({"out": z(3, 4, 68)[..., :64]}, ValueError, "16-byte boundaries"),
])
def test_refused_decodes(change, error, match):
    with pytest.raises(error, match=match):
        decode(**change)


def test_refused_places_of_out():
    buf = z(4, 4, 64)
    with pytest.raises(ValueError, match="q itself or lie apart"):
        decode(q=buf[:3], out=buf[1:])
    with pytest.raises(ValueError, match="on a CUDA/HIP device"):
        decode(q=buf[:3], out=buf[:3])
    k = z(6, 2, 16, 64)
    with pytest.raises(ValueError, match="apart from the caches"):
        decode(k_cache=k, out=k.view(-1, 4, 64)[:3])


@pytest.mark.parametrize("change,error,match", [
    ({"k": z(5, 2, 64, dtype=torch.float32)}, ValueError, "k must be bfloat16"),
    ({"k": 3}, TypeError, "k must be torch.Tensor"),
    ({"k": z(5, 3, 64)}, ValueError, "k must be \\[N, 2, 64\\]"),
    ({"v": z(5, 128)}, ValueError, "v must be \\[N, 2, 64\\]"),
    ({"v": z(4, 2, 64)}, ValueError, "same number of tokens"),
    ({"k": z(5, 2, 72)[..., 4:68]}, ValueError, "16-byte boundaries"),
    ({"slots": z(5, dtype=torch.int64)}, ValueError, "slots must be int32"),
    ({"slots": z(4, dtype=I32)}, ValueError, "one entry per token"),
    ({"slots": z(10, dtype=I32)[::2]}, ValueError, "slots must be contiguous"),
    ({"v": z(5, 2, 64).requires_grad_()}, ValueError, "requires grad"),
    ({"k_cache": z(1, 2, 16, 64).expand(6, 2, 16, 64)}, ValueError, "must not share memory"),
    ({**good(True), "v_scale": z(6, 1, 16, dtype=torch.float32).expand(6, 2, 16)}, ValueError, "must not share memory"),
])
def test_refused_writes(change, error, match):
    with pytest.raises(error, match=match):
        write(**change)


def test_refused_sources_and_places_in_the_cache():
    c = good()
    with pytest.raises(ValueError, match="apart from the caches"):
        write(**c, k=c["k_cache"].view(-1, 2, 64)[:5])
    with pytest.raises(ValueError, match="apart from the caches"):
        read(**c, v=c["v_cache"].view(-1, 2, 64)[:5])


@pytest.mark.parametrize("change,error,match", [
    ({"slots": z(2, 3, dtype=I32)}, ValueError, "slots must be contiguous"),
    ({"slots": None}, ValueError, "slots must be int32"),
    ({"k": z(5, 2, 64, dtype=torch.float32)}, ValueError, "k must be bfloat16"),
    ({"k": z(6, 2, 64)}, ValueError, "one entry per token|same number of tokens"),
    ({"v": z(5, 1, 64).expand(5, 2, 64)}, ValueError, "must not share memory"),
])
def test_refused_reads(change, error, match):
    with pytest.raises(error, match=match):
        read(**change)


@pytest.mark.parametrize("args,kw,match", [
    (((),), {}, "positive numbers"), (((8, 0),), {}, "positive numbers"), (((5, 4),), {}, "multiple of 8"),
    (((136,),), {}, "at most 128"), (((8,),), {"frequencies": "x"}, "'axis' or 'shared'"),
    (((8,),), {"pairing": "x"}, "'halves' or 'adjacent'"), (((8,),), {"theta": 0.0}, "theta"),
    (((8,),), {"theta": math.inf}, "theta"), (((8,),), {"theta": math.nan}, "theta"),
])
def test_refused_ropes(args, kw, match):
    with pytest.raises(ValueError, match=match):
        ma.AxialRope(*args, **kw)


def test_refused_rotations():
    rope = ma.AxialRope((16, 16))
    q, k, p = z(2, 7, 3, 64), z(2, 7, 1, 64), z(2, 7, dtype=I32)
    with pytest.raises(ValueError, match="on a CUDA/HIP device"):
        rope(q, k, p, layout="bshd")
    with pytest.raises(ValueError, match="on a CUDA/HIP device"):
        rope(q, None, p.unsqueeze(1).expand(2, 2, 7), layout="bshd", inplace=True)
    for args, kw, error, match in (
            ((q, k, p), {"layout": "sbhd"}, ValueError, "layout"),
            ((q.float(), k, p), {}, ValueError, "q must be bfloat16"),
            ((q, 3, p), {}, TypeError, "k must be torch.Tensor"),
            ((q[0], k, p), {}, ValueError, "4-D"),
            ((z(2, 7, 3, 32), k, p), {}, ValueError, "head_dim"),
            ((q, z(2, 7, 1, 128), p), {}, ValueError, "head_dim"),
            ((q, z(2, 8, 1, 64), p), {}, ValueError, "q's batch and sequence"),
            ((q, z(1, 7, 1, 64), p), {}, ValueError, "q's batch and sequence"),
            ((q, z(2, 7, 0, 64), p), {}, ValueError, "at least one head"),
            ((q, k, p.long()), {}, ValueError, "positions must be int32"),
            ((q, k, p[:1]), {}, ValueError, "positions must be"),
            ((q, k, p[:, :6]), {}, ValueError, "positions must be"),
            ((q, k, p.unsqueeze(1)), {}, ValueError, "positions must be"),
            ((z(2, 7, 3, 68)[..., :64], k, p), {}, ValueError, "16-byte boundaries"),
            ((q, z(2, 7, 1, 128)[..., ::2], p), {}, ValueError, "last dim"),
            ((z(2, 7, 1, 64).expand(2, 7, 3, 64), k, p), {"inplace": True}, ValueError, "must not share memory"),
            ((q, q, p), {"inplace": True}, ValueError, "must not share elements"),
            ((q, q[:, :, 1:], p), {"inplace": True}, ValueError, "must not share elements"),
            ((z(2, 7, 3, 64).requires_grad_(), k, p), {}, ValueError, "requires grad"),
            ((z(2, 7, 3, 128), z(2, 7, 3, 128).requires_grad_(), p), {}, ValueError, "requires grad")):
        with pytest.raises(error, match=match):
            rope(*args, **{"layout": "bshd", **kw})
    with pytest.raises(ValueError, match="head_dim"):
        ma.AxialRope((40,))(q, k, p[:1], layout="bshd")
    fused = z(2, 7, 6, 64)
    with pytest.raises(ValueError, match="on a CUDA/HIP device"):
        rope(fused[:, :, :3], fused[:, :, 3:5], p, layout="bshd", inplace=True)
    with pytest.raises(ValueError, match="must not share elements"):
        rope(fused[:, :, :4], fused[:, :, 3:5], p, layout="bshd", inplace=True)


def _shares(q, k):
    """Whether two views of one storage have an element in common, by enumeration."""
    at = []
    for t in (q, k):
        i = torch.tensor(t.storage_offset())
        for n, s in zip(t.shape, t.stride()):
            i = i[..., None] + torch.arange(n) * s
        at.append(set(i.flatten().tolist()))
    return bool(at[0] & at[1])


def test_views_that_are_written_together():
    """Whatever views pass for sharing nothing do share nothing."""
    g = torch.Generator().manual_seed(1)
    ri = lambda lo, hi: int(torch.randint(lo, hi, (1,), generator=g))  # noqa: E731
    base, passed = torch.zeros(4000, dtype=BF), 0
    for _ in range(3000):
        H, rowlen = ri(1, 5), 8 * ri(1, 9)
        views = []
        for _ in range(2):
            shape = (ri(1, 3), ri(1, 5), ri(1, H + 1), 8)
            views.append(base.as_strided(shape, (rowlen * 5, rowlen, 8, 1) if ri(0, 4) else (8 * ri(0, 60), 8 * ri(0, 9), 8, 1),
                                         8 * ri(0, 12)))
        if _checks.share_none(*views):
            passed += 1
            assert not _shares(*views), [(v.shape, v.stride(), v.storage_offset()) for v in views]
    assert passed > 100
    # Steps that do not nest: the second view's rows lie between the first's, and on some.
    lo, hi = (base.as_strided((2, 2, 1, 8), (120, 80, 8, 1), at) for at in (0, 40))
    _checks.one_place_each(lo, "lo", "who")
    assert _shares(lo, hi) and not _checks.share_none(lo, hi)


@pytest.mark.parametrize("shape,dim,order", [((2, 6, 2, 16, 64), 0, None), ((6, 2, 2, 16, 64), 1, None),
                                             ((6, 16, 2, 2, 64), 2, (0, 2, 1, 3)), ((6, 16, 2, 2, 64), 3, (0, 2, 1, 3)),
                                             ((6, 2, 16, 128), None, None)])
def test_caches_in_one_tensor(shape, dim, order):
    """K and V as slices of one tensor are written; one over the other is refused."""
    x = z(*shape)
    k, v = (x[..., :64], x[..., 64:]) if dim is None else (x.select(dim, 0), x.select(dim, 1))
    if order:
        k, v = k.permute(order), v.permute(order)
    with pytest.raises(ValueError, match="on a CUDA/HIP device"):
        write(k_cache=k, v_cache=v)
    for a, b in ((k, k), (v, v), (k[1:], k[:-1])):
        with pytest.raises(ValueError, match="must not share memory"):
            write(k_cache=a, v_cache=b)


def test_results_in_one_place():
    x = z(5, 2, 2, 64)
    with pytest.raises(ValueError, match="on a CUDA/HIP device"):
        read(k=x[:, 0], v=x[:, 1])
    with pytest.raises(ValueError, match="must not share memory"):
        read(k=x[:, 0], v=x[:, 0])
    c = good(True)
    with pytest.raises(ValueError, match="must not share memory"):
        write(**{**c, "v_scale": c["k_scale"]})
    with pytest.raises(ValueError, match="on a CUDA/HIP device"):  # read alone, they may be one
        decode(**{**c, "v_cache": c["k_cache"], "v_scale": c["k_scale"]})


def test_memory_checks_of_views():
    g = torch.Generator().manual_seed(2)
    base = torch.zeros(5000)
    for _ in range(500):
        shape = [int(torch.randint(1, 5, (1,), generator=g)) for _ in range(3)]
        stride = [int(torch.randint(0, 30, (1,), generator=g)) for _ in range(3)]
        t = base.as_strided(shape, stride, 3)
        at = [3 + sum(i * s for i, s in zip(x, stride)) for x in __import__("itertools").product(*map(range, shape))]
        a, b = _checks.extent(t)
        assert ((a - base.data_ptr()) // 4, (b - base.data_ptr()) // 4) == (min(at), max(at) + 1)
        try:
            _checks.one_place_each(t, "t", "who")
        except ValueError:
            continue
        assert len(set(at)) == len(at)


def test_launcher_codes():
    lib, n = _lib.lib, None
    st = (ctypes.c_longlong * 17)()
    p = ctypes.c_void_p(16)  # never followed: every call ends at a check or has no work
    dec = lambda B=1, T=1, Hq=4, Hkv=2, D=64, nb=1, page=16, w=1, x=p, ks=n, vs=n, s=st, ws=n: (  # noqa: E731
        lib.launch_gqa_decode_paged(x, p, p, ks, vs, p, n, p, p, B, T, Hq, Hkv, D, nb, page, w, s, 1.0, ws, n))
    assert dec(D=80) == -2 and dec(Hkv=0) == -3 and dec(Hq=5) == -3 and dec(Hq=1) == -3
    assert dec(B=-1) == -4 and dec(T=0) == -4 and dec(T=9) == -4 and dec(page=8) == -5 and dec(page=24) == -5
    assert dec(Hq=1 << 17) == -3 and dec(w=1 << 27) == -11
    assert dec(w=0) == -11 and dec(nb=0) == -11 and dec(x=n) == -6 and dec(ks=p) == -6 and dec(vs=p) == -6
    assert dec(s=None) == -6 and dec(w=1000) == -6  # a split without a workspace
    far = (ctypes.c_longlong * 17)()
    far[8] = (1 << 26) + 1
    assert dec(s=far) == -9
    assert dec(B=0) == 0
    # Sizes that no launch takes, past 31 bits in products of two or three of them.
    assert dec(B=1 << 30, Hq=16, Hkv=8, ws=p) == -8 and dec(B=1 << 16, Hq=1 << 16, Hkv=1 << 16, w=1000, ws=p) == -8
    assert lib.moonmath_gqa_decode_workspace(1 << 30, 1, 16, 8, 64, 16, 1000, 0, st) == 0
    for fn, order in ((lib.launch_gqa_kv_write, lambda k, ks: (k, p, p, p, ks, n, p)),
                      (lib.launch_gqa_kv_read, lambda k, ks: (p, p, ks, n, p, k, p))):
        run = lambda N=1, H=1, D=64, nb=1, page=16, k=p, ks=n, s=st: fn(*order(k, ks), N, H, D, nb, page, s, n)  # noqa: E731
        assert run(D=32) == -2 and run(H=0) == -3 and run(N=-1) == -4 and run(page=20) == -5 and run(nb=-1) == -11
        assert run(nb=1 << 28) == -11 and run(k=n) == -6 and run(ks=p) == -6 and run(s=None) == -6
        assert run(N=1 << 40) == -8 and run(N=1 << 31) == -8 and run(N=0) == 0
    rope = lambda B=1, S=1, Hq=1, Hk=0, D=64, P=8, A=1, q=p, s=st: (  # noqa: E731
        lib.launch_rope_axes(q, n, p, n, p, p, p, B, S, Hq, Hk, D, P, A, 0, 0, s, n))
    assert rope(D=32) == -2 and rope(Hq=0) == -3 and rope(Hk=-1) == -3 and rope(B=-1) == -4 and rope(S=-1) == -4
    assert rope(P=4) == -5 and rope(P=12) == -5 and rope(P=40) == -5 and rope(A=0) == -5
    assert rope(q=n) == -6 and rope(Hk=1) == -6 and rope(s=None) == -6 and rope(S=0) == 0 and rope(B=0) == 0
    assert rope(B=1 << 10, S=1 << 20) == -8


def test_workspace():
    """Records depend on the call's shape and not on its lengths; short contexts, empty
    batches and sizes that are refused need none."""
    heads, tokens = ((ctypes.c_longlong * 17)(*[0] * 6, *x) for x in ((1 << 20, 1 << 13, 128), (1 << 16, 128, 1024)))
    ws = lambda B, D=128, w=128, s=heads: _lib.lib.moonmath_gqa_decode_workspace(B, 1, 32, 8, D, 64, w, 0, s)  # noqa: E731
    assert ws(64, w=2) == 0 and ws(0) == 0 and ws(1, D=96) == 0 and ws(1, s=None) == 0
    for s in (heads, tokens):
        sizes = [ws(B, s=s) for B in (1, 4, 64, 1024)]
        assert 0 < sizes[0] <= sizes[1] <= sizes[2] <= sizes[3] <= sizes[2] + (16 << 10) < 64 << 20


HEADS, TOKENS = ((ctypes.c_longlong * 17)(*[0] * 6, *x) for x in ((1 << 20, 1 << 13, 128), (1 << 16, 128, 1024)))


def split(lens, q_len, Hq, Hkv, D, page, width, fp8, strides):
    n = len(lens)
    arr = (ctypes.c_int * max(n, 1))(*lens)
    args = (n, arr, q_len, Hq, Hkv, D, page, width, int(fp8), strides)
    count = _lib.lib.moonmath_gqa_decode_split(*args, None, 0)
    out = (ctypes.c_int * (8 * max(count, 1)))()
    assert _lib.lib.moonmath_gqa_decode_split(*args, out, count) == count
    return [tuple(out[8 * i:8 * i + 8]) for i in range(count)]


@pytest.mark.parametrize("seed", range(60))
def test_every_step_is_taken_once(seed):
    """The shares of random batches: each task's steps once and in order, at most one
    record of each kind for a workgroup, and the joined workgroups all hold a part; no
    workgroup has over twice the mean's steps, a task's own cost and a round more."""
    g = torch.Generator().manual_seed(seed)
    ri = lambda lo, hi: int(torch.randint(lo, hi, (1,), generator=g))  # noqa: E731
    B = [1, 2, 7, 64, 300, 700][ri(0, 6)]
    top = [40, 700, 5000, 70000][ri(0, 4)] if B <= 64 else [40, 700, 3000][ri(0, 3)]
    lens = [0 if ri(0, 9) == 0 else ri(1, top) for _ in range(B)]
    q_len, (Hq, Hkv) = ri(1, 9), [(8, 1), (4, 2), (16, 16), (32, 8), (48, 1), (24, 3)][ri(0, 6)]
    D, fp8, strides = [64, 128, 256][ri(0, 3)], bool(ri(0, 2)), [HEADS, TOKENS][ri(0, 2)]
    width = max(max(lens) // 16 + ri(1, 50), 100)
    parts = split(lens, q_len, Hq, Hkv, D, 16, width, fp8, strides)
    if not any(lens):
        assert parts == []
        return
    tasks = {}
    for p in parts:
        tasks.setdefault(p[1:3], []).append(p)
    per = len({t for _, t in tasks})
    assert len(tasks) == per * sum(n > 0 for n in lens) and per >= 1
    records, load = set(), {}
    for (b, _), group in tasks.items():
        steps = -(-lens[b] // 32)
        assert group[0][3] == 0 and group[-1][4] == steps and all(p[7] == steps for p in group)
        assert all(x[4] == y[3] and x[0] + 1 == y[0] for x, y in zip(group, group[1:]))
        assert all(p[3] < p[4] for p in group)
        if len(group) == 1:
            assert group[0][5] == -1 and group[0][6] == -1
            continue
        first = group[0][0]
        assert [p[5] for p in group] == [2 * first + 1] + [2 * p[0] for p in group[1:]]
        assert [p[6] for p in group] == [-1] * (len(group) - 1) + [first]
        assert not records & {p[5] for p in group}
        records |= {p[5] for p in group}
    for p in parts:
        load[p[0]] = load.get(p[0], 0) + p[4] - p[3]
    order = [p[0] for p in parts]
    assert order == sorted(order) and order[0] >= 0 and order[-1] < 512
    mean = sum(-(-n // 32) + 12 for n in lens if n) * per / min(512, max(order) + 1)
    assert max(load.values()) <= 2 * mean + 20


def test_split_codes():
    f, n, st = _lib.lib.moonmath_gqa_decode_split, (ctypes.c_int * 1)(5), HEADS
    assert f(1, n, 1, 4, 2, 80, 16, 1, 0, st, None, 0) == -2 and f(1, None, 1, 4, 2, 64, 16, 1, 0, st, None, 0) == -6
    assert f(1, n, 1, 4, 2, 64, 16, 1, 0, None, None, 0) == -6 and f(1, n, 1, 4, 2, 64, 16, 1000, 0, st, None, 4) == -6
    assert f(0, n, 1, 4, 2, 64, 16, 1000, 0, st, None, 0) == 0 and f(1, n, 1, 4, 2, 64, 16, 1, 0, st, None, 0) == 0


def test_native_path_leaves_cpu_calls():
    c, q = _lib.calls, z(1, 2, 64)
    assert c.gqa_write(q, q, q, q, q, None, None) is None and c.gqa_read(q, q, q, None, None, None, None) is None
    assert c.gqa_decode(q, q, q, q, q, None, None, None, None, False) is None
    assert c.rope(q, q, q, q, q, 1, "bhsd", True, False, False) is None and c.rope(1) is None


# ---- the oracle ----------------------------------------------------------------------------


@pytest.mark.parametrize("fp8", [False, True])
def test_oracle_decode_is_attention(fp8):
    """Against torch's attention in 64 bits with an explicit mask, and closed forms."""
    lens, T, page = [37, 1, 0, 16], 3, 16
    k, v, ks, vs = cache(9, 2, page, 64, fp8, 3)
    table = tables(lens, page, 9, 3)
    q = torch.randn(4, T, 6, 64, generator=torch.Generator().manual_seed(4)).to(BF)
    out, lse, bound, _ = og.decode(q, k, v, lens, table, None, ks, vs)
    for b, n in enumerate(lens):
        for t in range(T):
            m = n - T + t + 1
            if m <= 0:
                assert (out[b, t] == 0).all() and (lse[b, t] == -math.inf).all()
                continue
            rows = []
            for x, s in ((k, ks), (v, vs)):
                x = x.float() if s is None else x.float() * s[..., None]
                rows.append(torch.stack([x[table[b, i // page], :, i % page] for i in range(m)], 1).double())
            kk, vv = (r.repeat_interleave(3, 0) for r in rows)
            want = torch.nn.functional.scaled_dot_product_attention(q[b, t].double()[:, None], kk, vv)[:, 0]
            # the rows of an fp8 cache are formed in fp32 here
            assert torch.allclose(out[b, t], want, atol=1e-6, rtol=1e-6)
            if m == 1:
                assert torch.allclose(out[b, t], vv[:, 0], atol=1e-6)
    assert (bound >= 0).all()


def test_the_bound_sees_a_lost_token():
    """A token missing from the sum, or two exchanged in V, is outside the bound."""
    k, v, _, _ = cache(16, 1, 64, 64, False, 5)
    table = tables([1000], 64, 16, 5)
    q = torch.randn(1, 1, 4, 64, generator=torch.Generator().manual_seed(6)).mul(2).to(BF)
    out, _, bound, _ = og.decode(q, k, v, [1000], table)
    less, _, _, _ = og.decode(q, k, v, [999], table)
    v2 = v.clone()
    v2[table[0, 3], 0, 5], v2[table[0, 3], 0, 6] = v[table[0, 3], 0, 6], v[table[0, 3], 0, 5]
    other, _, _, _ = og.decode(q, k, v2, [1000], table)
    assert ((out - less).abs() > bound).any() and ((out - other).abs() > bound).any()


def test_oracle_quantize():
    codes, scale = og.quantize(torch.tensor([[448.0, -224.0, 1.0, 0.0], [0.0, 0.0, 0.0, 0.0], [2.0, math.nan, math.inf, -1.0]]).to(BF))
    assert scale.tolist() == [1.0, 2.0 ** -126, torch.tensor(2.0 / 448).item()]
    x = codes.float()
    assert x[0].tolist() == [448.0, -224.0, 1.0, 0.0] and x[1].tolist() == [0.0] * 4
    assert x[2, 0] == 448.0 and x[2, 1].isnan() and x[2, 2].isnan() and x[2, 3] == -224.0


def test_oracle_rope():
    """A turn of one radian per position, lengths kept, and neighbours or halves as pairs."""
    x = torch.randn(1, 2, 1, 64, generator=torch.Generator().manual_seed(7)).double()
    pos = torch.tensor([[[0, 3]]], dtype=I32)
    for pairing in ("halves", "adjacent"):
        y = og.rope(x, pos, (8,), 10000.0, "axis", pairing)
        i, j = (0, 8) if pairing == "halves" else (0, 1)
        assert torch.equal(y[0, 0], x[0, 0]) and torch.equal(y[..., 16:], x[..., 16:])
        a, b = x[0, 1, 0, i], x[0, 1, 0, j]
        assert torch.allclose(y[0, 1, 0, i], a * math.cos(3) - b * math.sin(3))
        assert torch.allclose(y[0, 1, 0, j], a * math.sin(3) + b * math.cos(3))
        assert torch.allclose(y.norm(), x.norm())
        assert torch.allclose(og.rope(y, pos, (8,), 10000.0, "axis", pairing, True), x)
