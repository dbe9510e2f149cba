"""Timed cases of the operators that serve a target model from its paged cache.

Three operators: `append` (norm and rotary position of a ragged batch's new q and
k, and the write of its k and v into the cache's pages, in 16 bits or quantised to
e4m3), `read` (rows of the cache back out of its pages) and `attention` (the new
tokens of a ragged batch against the paged cache). Each case runs either the
framework's entry points (`own`) or the same mathematics in elementary torch
operations.

Page order. A pool is [pages, kv heads, 16, head dim]; with layout "umma" the 16
rows of a (page, head) are stored as [2 groups of 8 rows][chunks of 16 bytes]
[8 rows][16 bytes], with "hnd" as plain rows. An e4m3 pool has a scale byte e + 127
for each row and head: the row's values are byte * 2^e, with e the smallest integer
from -126 on for which the row's largest magnitude is at most 448 * 2^e.
"""
import random

import torch

own = False

PAGE = 16
_DTYPE = {"bf16": torch.bfloat16, "f16": torch.float16}


# ---------------------------------------------------------------------------
# Cases
# ---------------------------------------------------------------------------
def _attention(name, requests, new, prefix, heads, *, type="bf16", store="same", layout="umma",
               window=0, sinks=False):
    return {"name": name, "kind": "attention", "requests": requests, "new_lo": new[0],
            "new_hi": new[1], "prefix_lo": prefix[0], "prefix_hi": prefix[1],
            "q_heads": heads[0], "kv_heads": heads[1], "dim": heads[2], "type": type,
            "store": store, "layout": layout, "window": window, "sinks": sinks}


def _append(name, requests, new, prefix, heads, *, type="bf16", store="same", layout="umma",
            norm=True, rotary=128, interleaved=False, tail=0):
    return {"name": name, "kind": "append", "requests": requests, "new_lo": new[0],
            "new_hi": new[1], "prefix_lo": prefix[0], "prefix_hi": prefix[1],
            "q_heads": heads[0], "kv_heads": heads[1], "dim": heads[2], "type": type,
            "store": store, "layout": layout, "norm": norm, "rotary": rotary,
            "interleaved": interleaved, "tail": tail}


def _read(name, requests, rows, first, heads, *, type="bf16", store="same", layout="umma"):
    return {"name": name, "kind": "read", "requests": requests, "new_lo": rows[0],
            "new_hi": rows[1], "prefix_lo": first[0], "prefix_hi": first[1], "q_heads": heads[0],
            "kv_heads": heads[1], "dim": heads[2], "type": type, "store": store, "layout": layout}


def listed():
    big, wide = (32, 8, 128), (64, 8, 64)
    return [
        # one user, one token: latency of a short decode step
        _attention("token_one", 1, (1, 1), (999, 999), big),
        # batched serving: 64 requests of 512 to 8192 tokens, one new token each
        _attention("tokens_64", 64, (1, 1), (512, 8191), big),
        # the same from a cache in 8 bits
        _attention("tokens_64_e4m3", 64, (1, 1), (512, 8191), big, store="e4m3"),
        # drafted blocks of 16 tokens verified as one sequence each
        _attention("blocks_16", 16, (16, 16), (2048, 16384), big),
        # a whole prompt into an empty cache
        _attention("prompt_8192", 1, (8192, 8192), (0, 0), big),
        # chunked prompts of odd lengths in a sliding layer with sinks
        _attention("chunks_window", 6, (201, 1499), (0, 6001), wide, window=128, sinks=True),
        # the last chunk of a 32k prompt over an 8-bit cache
        _attention("chunk_32k_e4m3", 1, (2048, 2048), (30720, 30720), big, store="e4m3"),
        # one new token of 64 requests on its way into the cache
        _append("write_tokens_64", 64, (1, 1), (512, 8191), big),
        # prompts, part of the head rotated in interleaved pairs, far positions, a padded batch
        _append("write_prompts_part", 9, (7, 3001), (0, 120000), wide, type="f16", norm=False,
                rotary=32, interleaved=True, tail=5),
        # prompts into an 8-bit cache and back out of it
        _append("write_read_e4m3", 3, (2001, 6001), (0, 20000), big, store="e4m3"),
        # handing a 32k prefix of an 8-bit cache to code that takes plain rows
        _read("read_32k_e4m3", 1, (32768, 32768), (0, 0), big, store="e4m3"),
        # short pieces of many requests
        _read("read_pieces", 24, (1, 700), (0, 2000), big),
    ]


def _log(rng, lo, hi):
    """A whole number of lo..hi, spread over its logarithm."""
    return max(lo, min(hi, round(lo * (hi / lo) ** rng.random())))


def _range(rng, lo, hi):
    a, b = sorted((_log(rng, lo, hi), _log(rng, lo, hi)))
    return a, b


def draw(rng):
    heads = [(32, 8, 128), (64, 8, 64), (16, 2, 128), (8, 8, 128), (24, 8, 64), (40, 8, 128),
             (12, 4, 128), (8, 1, 128)]
    while True:
        h = rng.choice(heads)
        kind = rng.choice(["attention"] * 4 + ["append"] * 2 + ["read"])
        store = rng.choice(["same", "same", "e4m3"])
        type = "bf16" if store == "e4m3" else rng.choice(["bf16", "bf16", "f16"])
        layout = "umma" if store == "e4m3" else rng.choice(["umma", "umma", "hnd"])
        more = dict(type=type, store=store, layout=layout)
        if kind == "attention":
            regime = rng.choice(["tokens", "blocks", "prompts"])
            if regime == "tokens":
                requests, new, prefix = _log(rng, 1, 128), (1, rng.choice([1, 1, 4])), (1, 32768)
            elif regime == "blocks":
                requests, new, prefix = _log(rng, 1, 48), _range(rng, 4, 64), (16, 32768)
            else:
                requests, new, prefix = _log(rng, 1, 12), _range(rng, 65, 8192), (1, 30000)
            prefix = _range(rng, *prefix)
            if rng.random() < 0.15:
                prefix = (0, prefix[1] // 4)
            case = _attention("", requests, new, prefix, h, sinks=rng.random() < 0.3,
                              window=rng.choice([0, 0, 0, _log(rng, 16, 4096)]), **more)
        elif kind == "append":
            rotary = rng.choice([0, h[2], h[2], h[2] // 2, h[2] // 4])
            case = _append("", _log(rng, 1, 128), _range(rng, 1, 4096),
                           _range(rng, 1, 120000), h, norm=rng.random() < 0.5, rotary=rotary,
                           interleaved=rng.random() < 0.5, tail=rng.choice([0, 0, 3]), **more)
        else:
            case = _read("", _log(rng, 1, 64), _range(rng, 1, 32768), _range(rng, 1, 4000), h,
                         **more)
        del case["name"]
        n, p = _lengths(case)
        w = work(case)
        padded = len(n) * max(n) * (max(n) + max(p)) * h[0] if kind == "attention" else 0
        gathered = len(n) * (max(n) + max(p)) * h[1] * h[2] if kind == "attention" else 0
        if (w["bytes"] <= 1.1e9 and w["flops"] <= 5.4e11 and padded <= 2.2e9 and gathered <= 6e8
                and sum(n) + sum(p) <= 4e5):
            return case


def _lengths(case):
    """(new tokens, tokens before them) of each request, by the case alone."""
    r = random.Random(repr([case[k] for k in ("requests", "new_lo", "new_hi", "prefix_lo",
                                              "prefix_hi")]))
    new = [r.randint(case["new_lo"], case["new_hi"]) for _ in range(case["requests"])]
    before = [r.randint(case["prefix_lo"], case["prefix_hi"]) for _ in range(case["requests"])]
    return new, before


def _visible(n, p, window):
    """Pairs (new token, key) that a causal mask with this window leaves."""
    if not window:
        return n * p + n * (n + 1) // 2
    full = max(0, min(n, p + n - window))  # tokens whose window is full
    rest = n - full
    return full * window + rest * p + rest * (rest + 1) // 2


def work(case):
    n, p = _lengths(case)
    Hq, Hk, D = case["q_heads"], case["kv_heads"], case["dim"]
    row = Hk * (D + 1) if case["store"] == "e4m3" else Hk * D * 2  # a token's K (or V) in the cache
    tokens = sum(n)
    if case["kind"] == "attention":
        w = case["window"]
        keys = sum(min(a + b, w + a - 1) if w else a + b for a, b in zip(n, p))
        pairs = sum(_visible(a, b, w) for a, b in zip(n, p))
        return {"bytes": 2 * keys * row + tokens * Hq * (2 * D * 2 + 4),
                "flops": 4 * D * Hq * pairs}
    if case["kind"] == "append":
        flops = tokens * (Hq + Hk) * D * (4 * case["norm"] + 3 * (case["rotary"] > 0))
        b = tokens * D * 2 * (2 * Hq + 2 * Hk) + 2 * tokens * row + tokens * case["rotary"] * 4
        if case["store"] == "e4m3":  # and read back
            b += 2 * tokens * row + 2 * tokens * Hk * D * 2
            flops += 4 * tokens * Hk * D
        return {"bytes": b, "flops": max(1, flops)}
    return {"bytes": 2 * tokens * row + 2 * tokens * Hk * D * 2,
            "flops": 2 * tokens * Hk * D}


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------
def _to_pages(rows, chunk):
    """[..., 16, D] plain rows -> the umma order of their block, chunks of `chunk` values."""
    s = rows.shape
    return rows.view(*s[:-2], 2, 8, s[-1] // chunk, chunk).transpose(-3, -2).reshape(s)


def _two(e):
    """2^e in 32 bits, e in -126..127."""
    return ((e + 127) << 23).view(torch.float32)


def _exponent(rows):
    """The scale exponent of each row in 8 bits, [..., 1]: 448 is 0.875 * 2^9."""
    m, e = torch.frexp(rows.abs().amax(-1, keepdim=True))
    e = (e - 9 + (m > 0.875).to(torch.int32)).clamp(-126, 127)
    return torch.where(m == 0, torch.full_like(e, -126), e)


def _pool(case, pages, g, device):
    """A pool of `pages` random pages: (values, scale bytes or None)."""
    shape = (pages, case["kv_heads"], PAGE, case["dim"])
    x = torch.randn(shape, generator=g, device=device)
    if case["store"] == "same":
        return x.to(_DTYPE[case["type"]]), None
    e = _exponent(x)
    q = (x * _two(-e)).to(torch.float8_e4m3fn)
    # rows of other sizes than the quantised ones: move every row's exponent
    shift = torch.randint(-6, 4, e.shape, generator=g, device=device)
    scale = (e + shift + 127).clamp(1, 254).to(torch.uint8).squeeze(-1)
    return _to_pages(q.view(torch.uint8), 16).view(torch.float8_e4m3fn), scale


def prepare(case, seed):
    device = torch.device("cuda")
    g = torch.Generator(device=device).manual_seed(seed * 2 + 1)
    dtype = _DTYPE[case["type"]]
    Hq, Hk, D = case["q_heads"], case["kv_heads"], case["dim"]
    n, p = _lengths(case)
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device=device)  # noqa: E731
    starts, bounds = [0], [0]
    for a, b in zip(n, p):
        starts.append(starts[-1] + a)
        bounds.append(bounds[-1] + -(-(a + b) // PAGE))
    N = starts[-1]
    s = {"case": case, "tokens": N, "new": n, "before": p, "starts": ints(starts),
         "lengths": ints(p), "bounds": ints(bounds), "bounds_host": bounds,
         "longest": (max(n), max(a + b for a, b in zip(n, p))),
         "table": torch.randperm(bounds[-1], generator=g, device=device).to(torch.int32),
         "layout": "paged_" + case["layout"]}
    for x in "kv":
        s[x + "_pool"], s[x + "_scale"] = _pool(case, bounds[-1], g, device)
    if case["kind"] == "read":
        s["k_rows"] = torch.zeros(N, Hk, D, dtype=dtype, device=device)
        s["v_rows"] = torch.zeros_like(s["k_rows"])
    elif case["kind"] == "attention":
        s["q"] = torch.randn(N, Hq, D, generator=g, device=device).to(dtype)
        s["sinks"] = torch.randn(Hq, generator=g, device=device) if case["sinks"] else None
        if own:
            from d2sd_b200 import PagedAttentionPlan
            s["plan"] = PagedAttentionPlan(n, [a + b for a, b in zip(n, p)], Hq, Hk, D, device,
                                           window=case["window"] or None, page_offsets=bounds)
    else:
        total = N + case["tail"]
        # the projections' output: q, k and v of a token side by side
        qkv = (2 * torch.randn(total, (Hq + 2 * Hk) * D, generator=g, device=device)).to(dtype)
        q, k, v = qkv.split([Hq * D, Hk * D, Hk * D], dim=1)
        s["q"], s["k"], s["v"] = q.view(total, Hq, D), k.view(total, Hk, D), v.view(total, Hk, D)
        s["q_out"] = torch.zeros(total, Hq, D, dtype=dtype, device=device)
        w = lambda: (1 + 0.2 * torch.randn(D, generator=g, device=device)).to(dtype)  # noqa: E731
        s["q_weight"], s["k_weight"] = (w(), w()) if case["norm"] else (None, None)
        s["cos"] = s["sin"] = None
        if case["rotary"]:
            rot = case["rotary"]
            inv = 1e6 ** (-torch.arange(0, rot, 2, dtype=torch.float64, device=device) / rot)
            at = torch.arange(s["longest"][1], dtype=torch.float64, device=device)
            angle = at[:, None] * inv[None]
            s["cos"], s["sin"] = angle.cos().float(), angle.sin().float()
        if case["store"] == "e4m3":
            s["k_rows"] = torch.zeros(N, Hk, D, dtype=dtype, device=device)
            s["v_rows"] = torch.zeros_like(s["k_rows"])
    return s


# ---------------------------------------------------------------------------
# One pass
# ---------------------------------------------------------------------------
def run(s):
    return _RUN[s["case"]["kind"]](s)


def _place(s):
    """(request, position, page, slot) of every new token."""
    at = torch.arange(s["tokens"], device=s["table"].device)
    r = torch.searchsorted(s["starts"].long(), at, right=True) - 1
    pos = s["lengths"].long()[r] + at - s["starts"].long()[r]
    page = s["table"].long()[s["bounds"].long()[r] + pos // PAGE]
    return r, pos, page, pos % PAGE


def _blocks(pool, layout):
    """A pool seen as [pages, heads, 2, 8, chunks, chunk]: row slot = 8 * i2 + i3."""
    P, H, S, D = pool.shape
    if layout == "paged_hnd":
        return pool.view(P, H, 2, 8, 1, D)
    c = 16 // pool.element_size()
    return pool.view(P, H, 2, D // c, 8, c).transpose(3, 4)


def _rows(s, x, page, slot):
    """Rows of pool x at (page, slot), in 32 bits: [tokens, heads, dim]."""
    pool = s[x + "_pool"]
    raw = pool.view(torch.uint8) if pool.element_size() == 1 else pool
    rows = _blocks(raw, s["layout"])[page, :, slot // 8, slot % 8].flatten(-2)
    rows = rows.view(pool.dtype).float() if pool.element_size() == 1 else rows.float()
    if s[x + "_scale"] is not None:
        e = s[x + "_scale"][page, :, slot].to(torch.int32) - 127
        rows = rows * _two(e[..., None])
    return rows


def _append_run(s):
    case = s["case"]
    if own:
        from d2sd_b200 import ops
        ops.append_kv(s["k"], s["v"], s["k_pool"], s["v_pool"], s["layout"], s["table"],
                      s["bounds"], s["starts"], s["lengths"], k_scale=s["k_scale"],
                      v_scale=s["v_scale"], q=s["q"], q_out=s["q_out"], q_weight=s["q_weight"],
                      k_weight=s["k_weight"], eps=1e-6, cos=s["cos"], sin=s["sin"],
                      interleaved=case["interleaved"])
    else:
        N = s["tokens"]
        _, pos, page, slot = _place(s)
        q, k, v = s["q"][:N].float(), s["k"][:N].float(), s["v"][:N].float()
        if case["norm"]:
            q = q * torch.rsqrt(q.square().mean(-1, keepdim=True) + 1e-6) * s["q_weight"].float()
            k = k * torch.rsqrt(k.square().mean(-1, keepdim=True) + 1e-6) * s["k_weight"].float()
        if case["rotary"]:
            c, d = s["cos"][pos][:, None], s["sin"][pos][:, None]
            q, k = (_rotate(x, c, d, case["rotary"], case["interleaved"]) for x in (q, k))
        s["q_out"][:N] = q.to(s["q_out"].dtype)
        _write(s, "k", k, page, slot)
        _write(s, "v", v, page, slot)
    if case["store"] == "e4m3":
        return {"q": s["q_out"], **_read_run(s)}
    return {"q": s["q_out"], "k": s["k_pool"], "v": s["v_pool"]}


def _rotate(x, c, s, rot, interleaved):
    head, rest = x[..., :rot], x[..., rot:]
    if interleaved:
        a, b = head[..., 0::2], head[..., 1::2]
        turned = torch.stack([a * c - b * s, b * c + a * s], -1).flatten(-2)
    else:
        a, b = head[..., :rot // 2], head[..., rot // 2:]
        turned = torch.cat([a * c - b * s, b * c + a * s], -1)
    return torch.cat([turned, rest], -1)


def _write(s, x, rows, page, slot):
    pool = s[x + "_pool"]
    if s[x + "_scale"] is None:
        blocks = _blocks(pool, s["layout"])
        blocks[page, :, slot // 8, slot % 8] = rows.to(pool.dtype).view(
            len(page), rows.shape[1], *blocks.shape[-2:])
        return
    e = _exponent(rows)
    s[x + "_scale"][page, :, slot] = (e + 127).to(torch.uint8).squeeze(-1)
    blocks = _blocks(pool.view(torch.uint8), s["layout"])
    blocks[page, :, slot // 8, slot % 8] = (rows * _two(-e)).to(torch.float8_e4m3fn).view(
        torch.uint8).view(len(page), rows.shape[1], *blocks.shape[-2:])


def _read_run(s):
    if own:
        from d2sd_b200 import ops
        ops.read_kv(s["k_pool"], s["v_pool"], s["layout"], s["table"], s["bounds"], s["starts"],
                    s["lengths"], s["k_rows"], s["v_rows"], k_scale=s["k_scale"],
                    v_scale=s["v_scale"])
    else:
        _, _, page, slot = _place(s)
        s["k_rows"][:] = _rows(s, "k", page, slot).to(s["k_rows"].dtype)
        s["v_rows"][:] = _rows(s, "v", page, slot).to(s["v_rows"].dtype)
    return {"k_rows": s["k_rows"], "v_rows": s["v_rows"]}


def _attention_run(s):
    case = s["case"]
    if own:
        from d2sd_b200 import paged_attention
        out, lse = paged_attention(s["q"], s["k_pool"], s["v_pool"], s["layout"], s["table"],
                                   s["plan"], k_scale=s["k_scale"], v_scale=s["v_scale"],
                                   sinks=s["sinks"])
        return {"out": out, "lse": lse}
    Hq, Hk, D = case["q_heads"], case["kv_heads"], case["dim"]
    R, G, (n_max, kv_max), device = case["requests"], Hq // Hk, s["longest"], s["q"].device
    starts, before = s["starts"].long(), s["lengths"].long()
    new = starts[1:] - starts[:-1]
    # every request padded to the longest: keys [R, Hk, kv, D], queries [R, Hk, G * n, D]
    key = torch.arange(kv_max, device=device).expand(R, kv_max)
    inside = key < (before + new)[:, None]
    page = s["table"].long()[torch.where(inside, s["bounds"].long()[:-1, None] + key // PAGE, 0)]
    k = _rows(s, "k", page.flatten(), (key % PAGE).flatten()).view(R, kv_max, Hk, D).transpose(1, 2)
    v = _rows(s, "v", page.flatten(), (key % PAGE).flatten()).view(R, kv_max, Hk, D).transpose(1, 2)
    i = torch.arange(n_max, device=device)
    tok = (starts[:-1, None] + i).clamp(max=s["tokens"] - 1)
    q = s["q"][tok].float().view(R, n_max, Hk, G, D).permute(0, 2, 3, 1, 4).reshape(R, Hk, -1, D)
    score = torch.matmul(q, k.transpose(2, 3)) * D ** -0.5
    pos = before[:, None] + i
    seen = (key[:, None, :] <= pos[..., None]) & inside[:, None, :]
    if case["window"]:
        seen &= key[:, None, :] > pos[..., None] - case["window"]
    score = score.view(R, Hk, G, n_max, kv_max).masked_fill_(~seen[:, None, None], float("-inf"))
    top = score.amax(-1, keepdim=True)
    weight = score.sub_(torch.where(top.isinf(), torch.zeros_like(top), top)).exp_()
    total = weight.sum(-1, keepdim=True)
    out = torch.matmul(weight.view(R, Hk, G * n_max, kv_max), v).view(R, Hk, G, n_max, D)
    out = torch.where(total > 0, out / total, torch.zeros_like(out))
    lse = (top + total.log())[..., 0]
    if case["sinks"]:
        out = out * torch.sigmoid(lse - s["sinks"].view(1, Hk, G, 1))[..., None]
    # the tokens that there are, back in the batch's order
    at = torch.arange(s["tokens"], device=device)
    r = torch.searchsorted(starts, at, right=True) - 1
    i = at - starts[r]
    out = out.permute(0, 3, 1, 2, 4)[r, i].reshape(-1, Hq, D).to(s["q"].dtype)
    lse = (lse * 1.4426950408889634).permute(0, 3, 1, 2)[r, i].reshape(-1, Hq)
    return {"out": out, "lse": lse}


_RUN = {"append": _append_run, "read": _read_run, "attention": _attention_run}


# ---------------------------------------------------------------------------
# The definitions in 64 bits, request by request
# ---------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    Hq, Hk, D = case["q_heads"], case["kv_heads"], case["dim"]
    G, dev = Hq // Hk, s["table"].device
    order = _slot_order(case, D, dev)

    def cached(x, r, lo, hi):
        """Rows lo..hi-1 of request r, [hi - lo, heads, dim]."""
        b = s["bounds_host"]
        pages = s["table"][b[r] + lo // PAGE:b[r] + -(-hi // PAGE)].long()
        flat = s[x + "_pool"][pages].double().flatten(-2)  # [pages, heads, 16 * dim]
        rows = flat[..., order].unflatten(-1, (PAGE, D))
        if s[x + "_scale"] is not None:
            rows = rows * torch.pow(2.0, s[x + "_scale"][pages].double() - 127.0)[..., None]
        rows = rows.transpose(1, 2).reshape(-1, Hk, D)
        return rows[lo % PAGE:lo % PAGE + hi - lo]

    if case["kind"] == "read":
        ks = [cached("k", r, b, b + a) for r, (a, b) in enumerate(zip(s["new"], s["before"]))]
        vs = [cached("v", r, b, b + a) for r, (a, b) in enumerate(zip(s["new"], s["before"]))]
        return {"k_rows": torch.cat(ks), "v_rows": torch.cat(vs)}

    if case["kind"] == "append":
        N, at = s["tokens"], 0
        pos = torch.cat([torch.arange(b, b + a, device=dev) for a, b in zip(s["new"], s["before"])])
        done = {}
        for x in "qkv":
            y = s[x][:N].double()
            if case["norm"] and x != "v":
                y = y / (y.pow(2).mean(-1, keepdim=True) + 1e-6).sqrt() * s[x + "_weight"].double()
            if case["rotary"] and x != "v":
                half = case["rotary"] // 2
                i = torch.arange(half, device=dev)
                a, b = (2 * i, 2 * i + 1) if case["interleaved"] else (i, i + half)
                z = torch.complex(y[..., a], y[..., b]) * torch.complex(
                    s["cos"][pos].double(), s["sin"][pos].double())[:, None]
                y = y.clone()
                y[..., a], y[..., b] = z.real, z.imag
            done[x] = y
        q = s["q_out"].double()
        q[:N] = done["q"]
        if case["store"] == "e4m3":
            return {"q": q, "k_rows": _e4m3(done["k"]), "v_rows": _e4m3(done["v"])}
        back = torch.empty_like(order)
        back[order] = torch.arange(len(order), device=dev)
        pools = {}
        for x in "kv":
            pool = s[x + "_pool"].double().flatten(-2)[..., order].unflatten(-1, (PAGE, D))
            at = 0
            for r, (a, b) in enumerate(zip(s["new"], s["before"])):
                lo = s["bounds_host"][r]
                p = torch.arange(b, b + a, device=dev)
                pool[s["table"][lo + p // PAGE].long(), :, p % PAGE] = done[x][at:at + a]
                at += a
            pools[x] = pool.flatten(-2)[..., back].unflatten(-1, (PAGE, D))
        return {"q": q, **pools}

    out = torch.empty(s["tokens"], Hq, D, dtype=torch.float64, device=dev)
    lse = torch.empty(s["tokens"], Hq, dtype=torch.float64, device=dev)
    first = 0
    for r, (a, b) in enumerate(zip(s["new"], s["before"])):
        k, v = cached("k", r, 0, a + b), cached("v", r, 0, a + b)
        j = torch.arange(a + b, device=dev)
        step = max(1, int(2.5e8 // ((a + b) * G)))
        for lo in range(0, a, step):
            hi = min(a, lo + step)
            i = torch.arange(b + lo, b + hi, device=dev)[:, None]
            hide = j > i
            if case["window"]:
                hide |= j + case["window"] <= i
            for h in range(Hk):
                rows = s["q"][first + lo:first + hi, h * G:(h + 1) * G].double()
                z = (rows.transpose(0, 1) @ k[:, h].T) / D ** 0.5
                z = z.masked_fill(hide, float("-inf"))
                ln = torch.logsumexp(z, -1)
                o = (z - ln[..., None]).exp() @ v[:, h]
                if case["sinks"]:
                    o = o / (1 + (s["sinks"][h * G:(h + 1) * G].double()[:, None] - ln).exp())[..., None]
                out[first + lo:first + hi, h * G:(h + 1) * G] = o.transpose(0, 1)
                lse[first + lo:first + hi, h * G:(h + 1) * G] = (ln / torch.log(
                    torch.tensor(2.0, dtype=torch.float64))).T
        first += a
    return {"out": out, "lse": lse}


def _slot_order(case, D, dev):
    """Where in a (page, head) block of 16 * D values element (slot, d) sits."""
    slot, d = torch.meshgrid(torch.arange(PAGE), torch.arange(D), indexing="ij")
    if case["layout"] == "hnd":
        return (slot * D + d).flatten().to(dev)
    c = 16 if case["store"] == "e4m3" else 8
    return (((slot // 8) * (D // c) + d // c) * 8 * c + (slot % 8) * c + d % c).flatten().to(dev)


def _e4m3(x):
    """What rows x stand for once they are held in 8 bits with a power-of-two scale."""
    two = 2.0 ** torch.arange(-130, 130, dtype=torch.float64)  # exact on the CPU
    two = two.to(x.device)
    top = x.abs().amax(-1, keepdim=True)
    # index of the first power of two with top <= 448 * 2^e, from 2^-126 on
    scale = two[torch.searchsorted(448 * two, top).clamp(min=4)]
    y = x / scale
    # spacing of e4m3 values: 2^-3 of the power of two at or below, 2^-9 at the least
    below = two[(torch.searchsorted(two, y.abs(), right=True) - 1).clamp(min=130 - 6)]
    return torch.round(y / (below / 8)) * (below / 8) * scale
