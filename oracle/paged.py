"""The target's own tokens and its paged cache, in float64 on the CPU: page order,
8-bit rows, norm + rotary position, and attention of a ragged batch."""
from __future__ import annotations

import torch


def page_index(layout: str, D: int, itemsize: int) -> torch.Tensor:
    """[16, D] places of a page block's elements (one head) in its flat storage."""
    r, d = torch.meshgrid(torch.arange(16), torch.arange(D), indexing="ij")
    if layout != "paged_umma":
        return r * D + d
    c = 16 // itemsize
    return ((r // 8) * (D // c) + d // c) * 8 * c + (r % 8) * c + d % c


def block_rows(pool: torch.Tensor, layout: str) -> torch.Tensor:
    """A pool [pages, Hk, 16, D] (or [pages, 16, Hk, D] for paged_nhd) as plain rows
    [pages, Hk, 16, D], float64, without scales."""
    if layout == "paged_nhd":
        return pool.transpose(1, 2).double()
    P, H, S, D = pool.shape
    if layout == "paged_hnd":
        return pool.double()
    idx = page_index(layout, D, pool.element_size()).flatten()
    return pool.double().flatten(2)[..., idx].view(P, H, 16, D)


def cached_rows(pool, layout, pages, n, scale=None):
    """Positions 0..n-1 of a sequence whose pages are ``pages``: [n, Hk, D]."""
    rows = block_rows(pool.cpu()[pages], layout)
    if scale is not None:
        byte = scale.cpu()[pages].double()
        f = torch.where(byte == 255, torch.full_like(byte, float("nan")),
                        torch.where(byte == 0, torch.zeros_like(byte), 2.0 ** (byte - 127)))
        rows = rows * f[..., None]
    return rows.transpose(1, 2).flatten(0, 1)[:n]


def e4m3_rows(x: torch.Tensor):
    """(values the rows stand for, scale bytes) of float64 rows [..., D]."""
    top = x.abs().amax(-1)
    e = torch.full_like(top, -126.0)
    for k in range(-126, 128):  # the smallest power of two that holds the row
        e = torch.where((top > 448 * 2.0 ** k), torch.full_like(e, k + 1.0), e)
    y = x / (2.0 ** e)[..., None]
    a = y.abs().clamp(min=2.0 ** -6)
    step = 2.0 ** (torch.floor(torch.log2(a)) - 3)
    step = torch.where(a >= 16 * step, 2 * step, step)  # log2 just below a power of two
    step = torch.where(a < 8 * step, step / 2, step)
    return torch.round(y / step) * step * (2.0 ** e)[..., None], (e + 127).to(torch.uint8)


def norm_rotate(x, weight, eps, cos, sin, positions, interleaved):
    """x [n, H, D] float64 -> RMSNorm (weight or None) and rotary position."""
    if weight is not None:
        x = x / torch.sqrt(x.square().mean(-1, keepdim=True) + eps) * weight.double()
    if cos is None:
        return x
    h = cos.shape[1]
    c, s = cos[positions].double()[:, None], sin[positions].double()[:, None]
    i = torch.arange(h)
    a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + h)
    y = x.clone()
    y[..., a] = x[..., a] * c - x[..., b] * s
    y[..., b] = x[..., b] * c + x[..., a] * s
    return y


def attention(q, k, v, *, causal=True, window=None, sinks=None, scale=None, sink_mode="exact"):
    """One request: q [n, Hq, D], k, v [kv, Hk, D] float64. Returns out, lse (base 2)
    and, for error bounds, sum_j p_j |v_j| and max_j scale * sum_d |q_d k_jd|."""
    n, Hq, D = q.shape
    kv, Hk, _ = k.shape
    G = Hq // Hk
    scale = D ** -0.5 if scale is None else scale
    kk, vv = k.repeat_interleave(G, 1), v.repeat_interleave(G, 1)
    s = torch.einsum("nhd,khd->hnk", q, kk) * scale
    size = (torch.einsum("nhd,khd->hnk", q.abs(), kk.abs()) * scale)
    i, j = torch.arange(n)[:, None] + kv - n, torch.arange(kv)[None]
    see = torch.ones(n, kv, dtype=torch.bool)
    if causal:
        see = j <= i
        if window is not None:
            see = see & (j > i - window)
    s = s.masked_fill(~see, float("-inf"))
    lse = torch.logsumexp(s, -1) if kv else torch.full((Hq, n), float("-inf"), dtype=torch.float64)
    p = torch.where(lse[..., None] == float("-inf"), torch.zeros_like(s), (s - lse[..., None]).exp())
    out = torch.einsum("hnk,khd->nhd", p, vv)
    absv = torch.einsum("hnk,khd->nhd", p, vv.abs())
    lse2 = lse / torch.log(torch.tensor(2.0, dtype=torch.float64))
    if sinks is not None:
        f = torch.sigmoid((lse if sink_mode == "exact" else lse2) - sinks.double()[:, None]).T[..., None]
        f = torch.where(f.isnan(), torch.zeros_like(f), f)
        out, absv = out * f, absv * f
    big = size.masked_fill(~see, 0.0).amax(-1) if kv else torch.zeros(Hq, n, dtype=torch.float64)
    return out, lse2.T, absv, big.T
