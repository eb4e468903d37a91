"""Seeded paged caches of grouped heads shared by the tests."""
import torch

from oracle import gqa as og

NAN = float("nan")


def cache(num_blocks, heads, page, D, fp8, seed, order="heads"):
    """K and V (and their scales): [nb, heads, page, D] views, on the CPU."""
    g = torch.Generator().manual_seed(seed)
    got = []
    for _ in range(2):
        x = torch.randn(num_blocks, heads, page, D, generator=g)
        x = (x * (0.25 + torch.rand(num_blocks, heads, page, 1, generator=g))).to(torch.bfloat16)
        s = None
        if fp8:
            x, s = og.quantize(x)
        if order == "tokens":
            x = x.transpose(1, 2).contiguous().transpose(1, 2)
        got.append((x, s))
    (k, ks), (v, vs) = got
    return k, v, ks, vs


def tables(lens, page, num_blocks, seed, width=None):
    """Random pages; entries past a request's pages are no block of the cache."""
    g = torch.Generator().manual_seed(seed + 1)
    need = [-(-max(n, 0) // page) for n in lens]
    assert sum(need) <= num_blocks
    perm = torch.randperm(num_blocks, generator=g).to(torch.int32)
    width = max(max(need), 1) if width is None else width
    table = torch.full((len(lens), width), -7, dtype=torch.int32)
    table[:, 1::2] = 2 ** 31 - 1
    at = 0
    for b, n in enumerate(need):
        n = min(n, width)
        table[b, :n] = perm[at:at + n]
        at += n
    return table


def poison(k, v, ks, vs, table, lens):
    """NaN and infinities in every row past a request's length within its last page, and
    in every block that no request holds."""
    nb, _, page, _ = k.shape
    used = torch.zeros(nb, page, dtype=torch.bool)
    for b, n in enumerate(lens):
        t = torch.arange(max(n, 0))
        used[table[b].long()[t // page], t % page] = True
    blk, row = (~used).nonzero(as_tuple=True)
    for i, x in enumerate((k, v)):
        if ks is None:
            x[blk, :, row] = torch.tensor([NAN, float("inf"), -float("inf")])[torch.arange(len(blk)) % 3][:, None, None].to(x.dtype)
        else:
            x.view(torch.uint8)[blk, :, row] = 0x7F
            (ks, vs)[i][blk, :, row] = torch.tensor([NAN, float("inf")])[torch.arange(len(blk)) % 2][:, None]
