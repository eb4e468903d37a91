"""Grouped-head paged cache, its decode attention and axial rotary positions, in
64 bits, from their definitions (torch on the CPU; no product code).

``decode`` also returns what its error bounds need; see ``decode_bound``.
"""
import math

import torch

U24 = 2.0 ** -24  # half a step of fp32
U8 = 2.0 ** -8    # half a step of bf16


def quantize(x):
    """bf16 rows [..., D] -> (e4m3fn codes, fp32 scales [...]): scale = fl32(max(amax
    / 448, 2^-126)) over the finite values, code = e4m3fn(fl32(x / scale)), NaN for
    what is not finite."""
    x = x.float()
    fine = x.isfinite()
    amax = torch.where(fine, x, 0.0).abs().amax(-1)
    scale = (amax / 448.0).clamp(min=2.0 ** -126)
    return torch.where(fine, x / scale[..., None], math.nan).to(torch.float8_e4m3fn), scale


def dequantize(codes, scale):
    """float64 values of codes [..., D] at scales [...] (None: bf16 rows as they are)."""
    x = codes.float().double()
    return x if scale is None else x * scale.double()[..., None]


def request_rows(cache, scale, table_row, n):
    """Tokens 0..n-1 of a request, float64 [Hkv, n, D]; cache [nb, Hkv, page, D]."""
    page = cache.shape[2]
    t = torch.arange(n)
    ids = table_row.long()[t // page].clamp(0, cache.shape[0] - 1)
    rows = cache.float().double()[ids, :, t % page]
    if scale is not None:
        rows = rows * scale.double()[ids, :, t % page][..., None]
    return rows.transpose(0, 1)


def decode(q, k_cache, v_cache, lens, table, scale=None, k_scale=None, v_scale=None):
    """q [B, T, Hq, D] -> (out, lse, bound) float64: bound is how far a bf16 output of
    the kernel may be from `out` (NaN or infinite where out is)."""
    B, T, Hq, D = q.shape
    Hkv, page = k_cache.shape[1], k_cache.shape[2]
    G = Hq // Hkv
    scale = D ** -0.5 if scale is None else scale
    out = torch.zeros(B, T, Hq, D, dtype=torch.float64)
    lse = torch.full((B, T, Hq), -math.inf, dtype=torch.float64)
    bound = torch.zeros_like(out)
    lse_bound = torch.zeros_like(lse)
    for b in range(B):
        S = min(max(int(lens[b]), 0), table.shape[1] * page)
        if S == 0:
            continue
        k = request_rows(k_cache, k_scale, table[b], S)
        v = request_rows(v_cache, v_scale, table[b], S)
        for t in range(T):
            n = S - T + t + 1
            if n <= 0:
                continue
            x = q[b, t].double().view(Hkv, G, D)
            s = torch.matmul(x, k[:, :n].transpose(1, 2)) * scale
            mag = torch.matmul(x.abs(), k[:, :n].abs().transpose(1, 2)) * abs(scale)
            l = torch.logsumexp(s, -1)
            p = torch.exp(s - l[..., None])
            p = torch.where((s == -math.inf) & (l[..., None] > -math.inf), 0.0, p)
            o = torch.matmul(p, v[:, :n])
            a = torch.matmul(p, v[:, :n].abs())
            # The kernel's errors, first order, u = 2^-24 (all sums in fp32):
            # a score: D products and D - 1 sums (D u mag), times scale * log2(e)
            # (itself rounded), the fp8 scale and the difference to the maximum
            # (5 u of values of at most mag + |m|, m the largest): e_s. exp2 adds 2 u
            # more, the split of p into two bf16 2^-16, V's fp8 scale u.
            mag = mag.where(s > -math.inf, torch.zeros((), dtype=torch.float64))
            worst = mag.amax(-1)
            e_s = (D * worst + 5 * 2 * worst) * U24
            e_p = e_s + 3 * U24 + 2.0 ** -16
            # The sums of p and of p v: at most n terms one after another, the rescales
            # and joins of fewer than n / 32 + 512 + 8 steps at 2 roundings each.
            e_sum = (n + 2 * (n // 32 + 520)) * U24
            rel = (2 * e_p + 2 * e_sum + 3 * U24)[..., None]
            out[b, t] = o.reshape(Hq, D)
            lse[b, t] = l.reshape(Hq)
            bound[b, t] = (U8 * o.abs() + rel * a * (1 + U8)).reshape(Hq, D) * 1.001
            # ln of the sum: the sum's error, the largest score's, and log2 and its product.
            lse_bound[b, t] = (e_s + e_sum + 4 * U24 * (1 + l.abs())).reshape(Hq)
    return out, lse, bound, lse_bound


def rope(x, positions, sections, theta, frequencies, pairing, inverse=False):
    """x [B, S, H, D] any float type, positions [axes, B, S] -> float64, each pair a
    complex number times e^(i angle)."""
    P = sum(sections)
    angles, done = [], 0
    for a, n in enumerate(sections):
        i = torch.arange(n, dtype=torch.float64)
        power = i / n if frequencies == "axis" else (done + i) / P
        angles.append(positions[a].double()[..., None] * theta ** -power)
        done += n
    angle = torch.cat(angles, -1)[:, :, None] * (-1.0 if inverse else 1.0)
    turn = torch.complex(angle.cos(), angle.sin())
    y = x.double().clone()
    if pairing == "adjacent":
        z = torch.view_as_complex(y[..., :2 * P].reshape(*y.shape[:-1], P, 2).contiguous()) * turn
        y[..., :2 * P] = torch.view_as_real(z).flatten(-2)
    else:
        z = torch.complex(y[..., :P].contiguous(), y[..., P:2 * P].contiguous()) * turn
        y[..., :2 * P] = torch.cat([z.real, z.imag], -1)
    return y


def rope_bound(x, positions, sections, theta, frequencies, pairing, inverse=False):
    """How far a bf16 result may be from ``rope``'s: half a step of bf16, and of the
    pair's magnitudes the cosine's and sine's errors (the number of turns in fp32, at
    most half a turn: 2^-26 of a turn = 2 pi 2^-26 rad; the functions 4 u; the angle
    itself in 64 bits: 3 roundings of |angle| 2^-53), a product and a sum (2 u)."""
    y = rope(x, positions, sections, theta, frequencies, pairing, inverse)
    P = sum(sections)
    x = x.double().abs()
    far = float(positions.abs().max()) if positions.numel() else 0.0
    err = 2 * math.pi * 2.0 ** -26 + 4 * U24 + 2 * U24 + 4 * far * 2.0 ** -53
    both = torch.zeros_like(x)
    if pairing == "adjacent":
        both[..., :2 * P] = (x[..., 0:2 * P:2] + x[..., 1:2 * P:2]).repeat_interleave(2, -1)
    else:
        both[..., :2 * P] = (x[..., :P] + x[..., P:2 * P]).repeat(1, 1, 1, 2)
    return y, U8 * y.abs() + 1.01 * err * both + 2.0 ** -133
