"""The operators of the target's own tokens on the GPU -- append, read, paged
attention, commit into an 8-bit cache -- against float64 (oracle/paged.py).

Error bounds, from the roundings the kernels make. Output o = sum p v / l: the
weights are rounded to the value type (at most u = finfo.eps / 2 relative each,
so u * sum p|v|), the output once more (u |o|); a score is an fp32 sum of D
products and a scale, off by at most (D + 4) 2^-24 sum|q k| scale, and the weights
by twice that relative to each other, with 2^-20 for the exponential and the fp32
sums of a row. A log-sum-exp is off by the score's error and 2^-20, times
log2 e."""
import numpy as np
import pytest
import torch

from oracle import paged as OP

pytestmark = pytest.mark.gpu

E4M3 = torch.float8_e4m3fn


def make_cache(g, kv_lens, Hk, D, dtype, layout, device, page_size=16, garbage=False):
    """Random cache of a ragged batch: pools (and scales) on the device, the page
    table, bounds, and every request's rows in float64."""
    pages = [-(-n // page_size) for n in kv_lens]
    bounds = [0]
    for p in pages:
        bounds.append(bounds[-1] + p)
    total = max(bounds[-1], 1) + 3
    table = torch.randperm(total, generator=g)[:max(bounds[-1], 1)].to(torch.int32)
    shape = (total, page_size, Hk, D) if layout == "paged_nhd" else (total, Hk, page_size, D)
    pools, scales = [], []
    for _ in range(2):
        x = torch.randn(shape, generator=g)
        if dtype == E4M3:
            vals, byte = OP.e4m3_rows(x.double() * 2.0 ** torch.randint(-5, 3, (*shape[:3], 1),
                                                                        generator=g))
            unit = vals / (2.0 ** (byte.double() - 127))[..., None]
            idx = OP.page_index(layout, D, 1).flatten()
            flat = torch.empty(total, Hk, 16 * D, dtype=torch.uint8)
            flat[..., idx] = unit.float().to(E4M3).view(torch.uint8).flatten(2)
            pools.append(flat.view(shape).view(E4M3))
            scales.append(byte)
        else:
            pools.append(x.to(dtype))
    rows = [[OP.cached_rows(p, layout, table[bounds[r]:bounds[r + 1]].long(), n,
                            scales[i] if scales else None) if page_size == 16 else
             OP.block_rows(p[table[bounds[r]:bounds[r + 1]].long()], layout).transpose(1, 2)
             .flatten(0, 1)[:n]
             for r, n in enumerate(kv_lens)] for i, p in enumerate(pools)]
    if garbage:  # NaN behind every request's last position, and in the pages nobody owns
        used = torch.zeros(total, page_size, dtype=torch.bool)
        for r, n in enumerate(kv_lens):
            pos = torch.arange(n)
            used[table[bounds[r]:bounds[r + 1]].long()[pos // page_size], pos % page_size] = True
        pg, sl = (~used).nonzero(as_tuple=True)
        for i, p in enumerate(pools):
            if dtype == E4M3:
                blk = p.view(torch.uint8).view(total, Hk, 2, D // 16, 8, 16)
                blk[pg, :, sl // 8, :, sl % 8] = 0x7f
                scales[i][pg, :, sl] = 255
            elif layout == "paged_umma":
                p.view(total, Hk, 2, D // 8, 8, 8)[pg, :, sl // 8, :, sl % 8] = float("nan")
            elif layout == "paged_nhd":
                p[pg, sl] = float("nan")
            else:
                p[pg, :, sl] = float("nan")
    to = lambda t: t.to(device)  # noqa: E731
    return dict(k=to(pools[0]), v=to(pools[1]), ks=to(scales[0]) if scales else None,
                vs=to(scales[1]) if scales else None, table=to(table), bounds=bounds,
                k_rows=rows[0], v_rows=rows[1], layout=layout)


def check_attention(out, lse, q, c, q_lens, D, dtype, **kw):
    u = torch.finfo(dtype).eps / 2
    at = 0
    for r, n in enumerate(q_lens):
        qr = q[at:at + n].double().cpu()
        o, l2, absv, big = OP.attention(qr, c["k_rows"][r], c["v_rows"][r], **kw)
        serr = (D + 4) * 2.0 ** -24 * big
        rel = (u + 2 * serr + 2.0 ** -20)[..., None]
        tol = rel * absv * (1 + u) + u * o.abs() + 1e-30
        got = out[at:at + n].double().cpu()
        assert not got.isnan().any(), r
        bad = (got - o).abs() - tol
        assert (bad <= 0).all(), (r, n, float((got - o).abs().max()), float(bad.max()))
        gl = lse[at:at + n].double().cpu()
        empty = l2 == float("-inf")
        assert torch.equal(gl == float("-inf"), empty), r
        if n:
            d = (gl - l2)[~empty].abs()
            t = ((serr + 2.0 ** -20) * 1.4427 + l2.abs() * 2.0 ** -23)[~empty]
            assert (d <= t).all(), (r, float(d.max()))
        at += n


# (q lengths, kv lengths): single tokens, lengths of zero, odd ones, pages that end
# inside a tile, rows without a key (kv < q), more than one tile and many splits
MIXED = ([1, 0, 5, 33, 2, 17, 3], [1, 40, 5, 130, 700, 17, 0])
CASES = [
    # Hq, Hk, D, type, store, layout, lens, window, sinks
    (32, 8, 128, "bf16", "same", "paged_umma", ([1] * 6, [1, 15, 16, 17, 128, 3001]), None, False),
    (32, 8, 128, "bf16", "same", "paged_umma", MIXED, None, False),
    (64, 8, 64, "bf16", "same", "paged_umma", MIXED, 20, True),
    (10, 2, 128, "f16", "same", "paged_umma", MIXED, None, True),
    (6, 2, 64, "f16", "same", "paged_hnd", MIXED, 129, False),
    (8, 8, 128, "bf16", "same", "paged_nhd", MIXED, None, False),
    (32, 8, 128, "bf16", "e4m3", "paged_umma", MIXED, None, False),
    (64, 8, 64, "bf16", "e4m3", "paged_umma", MIXED, 100, True),
    (16, 1, 128, "bf16", "e4m3", "paged_umma", ([3, 1], [5000, 257]), None, False),
    (32, 8, 128, "bf16", "same", "paged_umma", ([1], [20011]), None, False),
    (4, 1, 64, "bf16", "same", "paged_umma", ([300], [450]), None, False),
    (32, 8, 128, "bf16", "same", "paged_umma", ([257, 130], [257, 1000]), None, False),
    (32, 8, 128, "bf16", "same", "paged_umma", ([257, 130], [300, 1000]), 70, True),
    (40, 8, 128, "f16", "same", "paged_hnd", ([200], [333]), None, False),
    (12, 4, 128, "bf16", "e4m3", "paged_umma", ([190, 1], [700, 90]), 300, False),
    (128, 1, 64, "bf16", "same", "paged_umma", ([3, 40], [100, 41]), None, False),
    # many short units for each CTA, whose first and last key tiles are both cut
    (64, 8, 64, "bf16", "same", "paged_umma", ([1300, 900, 33], [1300, 2000, 300]), 128, True),
    (64, 8, 64, "bf16", "e4m3", "paged_umma", ([1300, 900, 33], [1300, 2000, 300]), 128, False),
    (32, 8, 128, "f16", "same", "paged_hnd", ([1000, 70], [1000, 500]), 50, False),
]
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16}


@pytest.mark.parametrize("i", range(len(CASES)))
@pytest.mark.parametrize("garbage", [False, True])
def test_attention(cuda_device, i, garbage):
    import d2sd_b200 as d
    Hq, Hk, D, t, store, layout, (ql, kl), window, with_sinks = CASES[i]
    dtype = TYPES[t]
    g = torch.Generator().manual_seed(100 + i)
    c = make_cache(g, kl, Hk, D, E4M3 if store == "e4m3" else dtype, layout, cuda_device,
                   garbage=garbage)
    n = sum(ql)
    # a strided view (the projection's output) and rows behind the last request
    q = torch.randn(n + 2, Hq + 3, D, generator=g).to(dtype).to(cuda_device)[:, 1:Hq + 1]
    sinks = torch.randn(Hq, generator=g).to(cuda_device) if with_sinks else None
    plan = d.PagedAttentionPlan(ql, kl, Hq, Hk, D, cuda_device, window=window,
                                page_offsets=c["bounds"],
                                cache_dtype=c["k"].dtype if garbage else None)
    out = torch.full((n + 2, Hq + 1, D), 7.0, dtype=dtype, device=cuda_device)[:, :Hq]
    lse = torch.full((n + 2, Hq), 7.0, device=cuda_device)
    for _ in range(2):  # the second call finds the workspace as the first left it
        d.paged_attention(q, c["k"], c["v"], layout, c["table"], plan, k_scale=c["ks"],
                          v_scale=c["vs"], sinks=sinks, out=out, lse=lse)
        check_attention(out, lse, q, c, ql, D, dtype, window=window,
                        sinks=None if sinks is None else sinks.cpu())
    assert (out[n:] == 7).all() and (lse[n:] == 7).all()
    assert int(plan.status) == 0


def test_attention_widens_the_span_of_long_chunks(cuda_device):
    """A chunk that goes over its 8-bit keys often enough to widen them first, between
    requests of single tokens whose pages lie around it."""
    import d2sd_b200 as d
    Hq, Hk, D, ql, kl = 16, 2, 128, [1, 300, 200, 1], [200, 310, 1000, 77]
    g = torch.Generator().manual_seed(21)
    c = make_cache(g, kl, Hk, D, E4M3, "paged_umma", cuda_device, garbage=True)
    q = torch.randn(sum(ql), Hq, D, generator=g).to(torch.bfloat16).to(cuda_device)
    plan = d.PagedAttentionPlan(ql, kl, Hq, Hk, D, cuda_device, page_offsets=c["bounds"])
    assert plan.widen and plan.wide_pages == c["bounds"][3] - c["bounds"][1]
    for _ in range(2):
        out, lse = d.paged_attention(q, c["k"], c["v"], "paged_umma", c["table"], plan,
                                     k_scale=c["ks"], v_scale=c["vs"])
        check_attention(out, lse, q, c, ql, D, torch.bfloat16)
    with pytest.raises(ValueError):  # a page table that ends inside the span
        d.paged_attention(q, c["k"], c["v"], "paged_umma", c["table"][:30], plan, k_scale=c["ks"],
                          v_scale=c["vs"])


@pytest.mark.parametrize("store", ["same", "e4m3"])
def test_attention_without_causal_mask(cuda_device, store):
    import d2sd_b200 as d
    Hq, Hk, D, ql, kl = 16, 4, 128, [4, 3, 50], [60, 0, 333]
    g = torch.Generator().manual_seed(5)
    c = make_cache(g, kl, Hk, D, E4M3 if store == "e4m3" else torch.bfloat16, "paged_umma",
                   cuda_device, garbage=True)
    q = torch.randn(sum(ql), Hq, D, generator=g).to(torch.bfloat16).to(cuda_device)
    plan = d.PagedAttentionPlan(ql, kl, Hq, Hk, D, cuda_device, causal=False,
                                page_offsets=c["bounds"])
    out, lse = d.paged_attention(q, c["k"], c["v"], "paged_umma", c["table"], plan, sm_scale=0.05,
                                 k_scale=c["ks"], v_scale=c["vs"])
    check_attention(out, lse, q, c, ql, D, torch.bfloat16, causal=False, scale=0.05)


@pytest.mark.parametrize("layout,page_size", [("paged_hnd", 32), ("paged_nhd", 64)])
def test_attention_larger_pages(cuda_device, layout, page_size):
    import d2sd_b200 as d
    Hq, Hk, D, ql, kl = 8, 2, 64, [2, 100], [77, 300]
    g = torch.Generator().manual_seed(6)
    c = make_cache(g, kl, Hk, D, torch.bfloat16, layout, cuda_device, page_size=page_size)
    q = torch.randn(sum(ql), Hq, D, generator=g).to(torch.bfloat16).to(cuda_device)
    plan = d.PagedAttentionPlan(ql, kl, Hq, Hk, D, cuda_device, page_offsets=c["bounds"])
    out, lse = d.paged_attention(q, c["k"], c["v"], layout, c["table"], plan)
    check_attention(out, lse, q, c, ql, D, torch.bfloat16)


def test_attention_large_scores(cuda_device):
    """Scores in the hundreds: the running maximum moves through the keys."""
    import d2sd_b200 as d
    Hq, Hk, D, ql, kl = 8, 2, 128, [1, 140], [2000, 900]
    g = torch.Generator().manual_seed(7)
    c = make_cache(g, kl, Hk, D, torch.bfloat16, "paged_umma", cuda_device)
    q = (20 * torch.randn(sum(ql), Hq, D, generator=g)).to(torch.bfloat16).to(cuda_device)
    plan = d.PagedAttentionPlan(ql, kl, Hq, Hk, D, cuda_device, page_offsets=c["bounds"])
    out, lse = d.paged_attention(q, c["k"], c["v"], "paged_umma", c["table"], plan)
    check_attention(out, lse, q, c, ql, D, torch.bfloat16)


@pytest.mark.parametrize("n", [1, 70])
def test_attention_reference_sink_mode(cuda_device, n):
    import d2sd_b200 as d
    Hq, Hk, D, kl = 8, 2, 64, [300]
    g = torch.Generator().manual_seed(30 + n)
    c = make_cache(g, kl, Hk, D, torch.bfloat16, "paged_umma", cuda_device)
    q = torch.randn(n, Hq, D, generator=g).to(torch.bfloat16).to(cuda_device)
    sinks = (4 + torch.randn(Hq, generator=g)).to(cuda_device)
    plan = d.PagedAttentionPlan([n], kl, Hq, Hk, D, cuda_device)
    out, lse = d.paged_attention(q, c["k"], c["v"], "paged_umma", c["table"], plan, sinks=sinks,
                                 sink_mode="reference")
    check_attention(out, lse, q, c, [n], D, torch.bfloat16, sinks=sinks.cpu(), sink_mode="reference")


def test_attention_of_no_tokens(cuda_device):
    import d2sd_b200 as d
    kp = torch.zeros(4, 2, 16, 64, dtype=torch.bfloat16, device=cuda_device)
    table = torch.arange(4, dtype=torch.int32, device=cuda_device)
    plan = d.PagedAttentionPlan([0, 0], [7, 0], 4, 2, 64, cuda_device, page_offsets=[0, 1])
    for n in (0, 3):
        q = torch.zeros(n, 4, 64, dtype=torch.bfloat16, device=cuda_device)
        out = torch.full_like(q, 2.0)
        d.paged_attention(q, kp, kp, "paged_umma", table, plan, out=out)
        assert (out == 2).all()


def test_attention_bad_page_ids(cuda_device):
    """Ids outside the pool are read as its first or last page: no fault, and the
    other requests' rows are right."""
    import d2sd_b200 as d
    Hq, Hk, D, ql, kl = 8, 2, 128, [1, 1, 150], [50, 64, 400]
    g = torch.Generator().manual_seed(8)
    c = make_cache(g, kl, Hk, D, torch.bfloat16, "paged_umma", cuda_device)
    c["table"][c["bounds"][1]] = 1 << 30
    c["table"][c["bounds"][1] + 1] = -5
    q = torch.randn(sum(ql), Hq, D, generator=g).to(torch.bfloat16).to(cuda_device)
    plan = d.PagedAttentionPlan(ql, kl, Hq, Hk, D, cuda_device, page_offsets=c["bounds"])
    out, lse = d.paged_attention(q, c["k"], c["v"], "paged_umma", c["table"], plan)
    for r, (a, b) in ((0, (0, 1)), (2, (2, 152))):
        one = dict(c, k_rows=[c["k_rows"][r]], v_rows=[c["v_rows"][r]])
        check_attention(out[a:b], lse[a:b], q[a:b], one, [ql[r]], D, torch.bfloat16)


def test_captured_call_replays_after_update(cuda_device):
    """A reserved plan: one captured call, other lengths at every replay."""
    import d2sd_b200 as d
    Hq, Hk, D = 16, 4, 128
    g = torch.Generator().manual_seed(9)
    full = [900, 300, 2500]
    c = make_cache(g, full, Hk, D, torch.bfloat16, "paged_umma", cuda_device)
    q = torch.randn(400, Hq, D, generator=g).to(torch.bfloat16).to(cuda_device)
    plan = d.PagedAttentionPlan([1, 1, 1], [9, 9, 9], Hq, Hk, D, cuda_device,
                                page_offsets=c["bounds"], reserve=(3, 400))
    out = torch.zeros_like(q)
    lse = torch.zeros(400, Hq, device=cuda_device)
    call = lambda: d.paged_attention(q, c["k"], c["v"], "paged_umma", c["table"], plan,  # noqa
                                     out=out, lse=lse)
    call()
    s = torch.cuda.Stream(cuda_device)
    s.wait_stream(torch.cuda.current_stream(cuda_device))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(s), torch.cuda.graph(graph, stream=s):
        call()
    torch.cuda.current_stream(cuda_device).wait_stream(s)
    for ql, kl in (([1, 1, 1], [9, 9, 9]), ([1, 1, 1], [900, 16, 2500]), ([40, 0, 350], [41, 7, 2400]),
                   ([0, 0, 0], [5, 5, 5]), ([1, 260, 1], [1, 290, 1])):
        plan.update(ql, kl, c["bounds"])
        graph.replay()
        torch.cuda.synchronize(cuda_device)
        cut = dict(c, k_rows=[x[:n] for x, n in zip(c["k_rows"], kl)],
                   v_rows=[x[:n] for x, n in zip(c["v_rows"], kl)])
        check_attention(out, lse, q, cut, ql, D, torch.bfloat16)
    with pytest.raises(ValueError):
        plan.update([4000] * 3, [4000] * 3, c["bounds"])
    del graph


def test_two_plans_on_two_streams(cuda_device):
    import d2sd_b200 as d
    Hq, Hk, D = 32, 8, 128
    g = torch.Generator().manual_seed(10)
    jobs = []
    for kl in ([4000], [3000]):
        c = make_cache(g, kl, Hk, D, torch.bfloat16, "paged_umma", cuda_device)
        q = torch.randn(1, Hq, D, generator=g).to(torch.bfloat16).to(cuda_device)
        jobs.append((c, q, d.PagedAttentionPlan([1], kl, Hq, Hk, D, cuda_device),
                     torch.cuda.Stream(cuda_device)))
    torch.cuda.synchronize(cuda_device)
    res = []
    for _ in range(5):
        for c, q, plan, s in jobs:
            with torch.cuda.stream(s):
                res.append(d.paged_attention(q, c["k"], c["v"], "paged_umma", c["table"], plan))
    torch.cuda.synchronize(cuda_device)
    for x, (o, l) in enumerate(res):
        c, q, _, _ = jobs[x % 2]
        check_attention(o, l, q, c, [1], D, torch.bfloat16)


# ---------------------------------------------------------------------------
# append, read, commit
# ---------------------------------------------------------------------------
APPEND = [
    # type, store, layout, Hq, Hk, D, norm, rotary, interleaved
    ("bf16", "same", "paged_umma", 32, 8, 128, True, 128, False),
    ("bf16", "same", "paged_umma", 64, 8, 64, False, 64, False),
    ("f16", "same", "paged_hnd", 6, 2, 64, True, 32, True),
    ("f32", "same", "paged_hnd", 4, 1, 128, True, 48, False),
    ("f32", "same", "paged_nhd", 4, 2, 64, False, 16, True),
    ("bf16", "same", "paged_nhd", 5, 5, 128, False, 0, False),
    ("bf16", "e4m3", "paged_umma", 32, 8, 128, True, 128, False),
    ("f16", "e4m3", "paged_umma", 8, 8, 64, False, 32, True),
    ("bf16", "e4m3", "paged_umma", 0, 3, 128, False, 0, False),
    ("bf16", "same", "paged_umma", 40, 8, 128, True, 96, False),
]
ALL_TYPES = dict(TYPES, f32=torch.float32)


def new_pool(total, Hk, D, dtype, layout, device, g):
    shape = (total, 16, Hk, D) if layout == "paged_nhd" else (total, Hk, 16, D)
    x = torch.randint(1, 100, shape, generator=g)
    if dtype == E4M3:
        return (x.to(torch.uint8).view(E4M3).to(device),
                torch.randint(100, 130, shape[:3], generator=g).to(torch.uint8).to(device))
    return x.to(dtype).to(device), None


@pytest.mark.parametrize("i", range(len(APPEND)))
def test_append_and_read(cuda_device, i):
    from d2sd_b200 import ops
    t, store, layout, Hq, Hk, D, norm, rot, inter = APPEND[i]
    dtype, dev = ALL_TYPES[t], cuda_device
    g = torch.Generator().manual_seed(40 + i)
    ql, first = [1, 0, 37, 16, 3], [0, 9, 5, 4000, 31]
    R, n = len(ql), sum(ql)
    starts, bounds = [0], [0]
    for a, b in zip(ql, first):
        starts.append(starts[-1] + a)
        bounds.append(bounds[-1] + -(-(a + b) // 16))
    total = bounds[-1] + 2
    table = torch.randperm(total, generator=g)[:bounds[-1]].to(torch.int32)
    kp, ks = new_pool(total, Hk, D, E4M3 if store == "e4m3" else dtype, layout, dev, g)
    vp, vs = new_pool(total, Hk, D, E4M3 if store == "e4m3" else dtype, layout, dev, g)
    k0, v0 = kp.clone(), vp.clone()
    # q, k, v side by side, two rows behind the last request; rows of many sizes
    size = 2.0 ** torch.randint(-12, 8, (n + 2, Hq + 2 * Hk, 1), generator=g)
    qkv = (torch.randn(n + 2, Hq + 2 * Hk, D, generator=g) * size).to(dtype)
    qkv[0, -1] = 0.0  # a row of zeros
    q, k, v = qkv[:, :Hq], qkv[:, Hq:Hq + Hk], qkv[:, Hq + Hk:]
    w = [(1 + 0.3 * torch.randn(D, generator=g)).to(dtype) if norm else None for _ in range(2)]
    cos = sin = None
    if rot:
        from d2sd_b200 import rope_tables
        cos, sin = rope_tables(4016, rot, 1e4, "cpu")
    dq = qkv.to(dev)
    up = lambda x: None if x is None else x.to(dev)  # noqa: E731
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    status = torch.zeros(1, dtype=torch.int32, device=dev)
    q_out = torch.full((n + 2, Hq, D), 3.0, dtype=dtype, device=dev) if Hq else None
    ops.append_kv(dq[:, Hq:Hq + Hk], dq[:, Hq + Hk:], kp, vp, layout, up(table), ints(bounds),
                  ints(starts), ints(first), k_scale=ks, v_scale=vs, q=dq[:, :Hq] if Hq else None,
                  q_out=q_out, q_weight=up(w[0]) if Hq else None, k_weight=up(w[1]), eps=1e-5,
                  cos=up(cos), sin=up(sin), interleaved=inter, status=status)
    assert int(status) == 0
    pos = torch.cat([torch.arange(b, b + a) for a, b in zip(ql, first)])
    f64 = lambda x: x[:n].double()  # noqa: E731
    want_k = OP.norm_rotate(f64(k), w[1], 1e-5, cos, sin, pos, inter)
    want_v = f64(v)
    # fp32 arithmetic: a norm of D squares and five products, (D / 2 + 16) 2^-24 of the pair's size
    u = torch.finfo(dtype).eps / 2
    fp32 = (D // 2 + 16) * 2.0 ** -24

    def pair(x):  # size of the rotated pair each element comes from (sqrt 2 of its own at most)
        return x.abs().amax(-1, keepdim=True) * 2 if rot else x.abs()
    if Hq:
        want_q = OP.norm_rotate(f64(q), w[0], 1e-5, cos, sin, pos, inter)
        err = (q_out[:n].double().cpu() - want_q).abs()
        tiny = torch.finfo(dtype).smallest_normal * u * 2
        assert (err <= u * want_q.abs() + fp32 * pair(want_q) + tiny).all()
        assert (q_out[n:] == 3).all()
    # read back
    out_t = torch.bfloat16 if store == "e4m3" and t == "bf16" else dtype
    kr = torch.full((n + 1, Hk, D), 5.0, dtype=out_t, device=dev)
    vr = torch.full((n + 1, Hk, D), 5.0, dtype=out_t, device=dev)
    ops.read_kv(kp, vp, layout, up(table), ints(bounds), ints(starts), ints(first), kr, vr,
                k_scale=ks, v_scale=vs, status=status)
    assert int(status) == 0 and (kr[n:] == 5).all() and (vr[n:] == 5).all()
    got_k, got_v = kr[:n].double().cpu(), vr[:n].double().cpu()
    if store == "e4m3":
        # e4m3: half a step is 2^-4 of the value, or of the smallest normal value
        # 2^-6 * 2^e where the row's scale 2^e is at most 2 * max / 448
        def bound(x):
            floor = x.abs().amax(-1, keepdim=True) * 2 / 448 * 2.0 ** -6 * 2.0 ** -4
            return torch.maximum(x.abs() * 2.0 ** -4, floor) + fp32 * pair(x)
        if t == "bf16":  # exact values, without rotation or norm the very ones
            assert torch.equal(got_v, OP.e4m3_rows(want_v)[0])
            assert ((got_k - want_k).abs() <= bound(want_k)).all()
            if not norm and not rot:
                assert torch.equal(got_k, OP.e4m3_rows(want_k)[0])
        else:  # read into fp16: small values are subnormal there
            extra = 2.0 ** -25
            assert ((got_v - want_v).abs() <= bound(want_v) * (1 + 2 ** -10) + extra).all()
            assert ((got_k - want_k).abs() <= bound(want_k) * (1 + 2 ** -10) + extra).all()
    else:
        tiny = torch.finfo(dtype).smallest_normal * u * 2
        assert torch.equal(got_v, want_v)
        assert ((got_k - want_k).abs() <= u * want_k.abs() + fp32 * pair(want_k) + tiny).all()
    # nothing else in the pools changed
    for new, old in ((kp, k0), (vp, v0)):
        a, b = (OP.block_rows(x.cpu(), layout) for x in (new, old))
        touched = torch.zeros(total, 16, dtype=torch.bool)
        req = torch.repeat_interleave(torch.arange(R), torch.tensor(ql))
        touched[table[torch.tensor(bounds)[req] + pos // 16].long(), pos % 16] = True
        keep = ~touched[:, None, :, None].expand_as(a)
        assert torch.equal(a[keep], b[keep])


def test_append_skips_bad_positions_and_pages(cuda_device):
    from d2sd_b200 import ops, rope_tables
    dev, Hk, D = cuda_device, 2, 64
    g = torch.Generator().manual_seed(3)
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    cos, sin = rope_tables(30, D, 1e4, dev)
    cases = [(4, [0, 3], [0, 2], [30], None),         # runs past the request's two pages
             (4, [0, 3], [0, 2], [-1], None),
             (5, [0, 1], [0, 1], [3], [77]),          # a page id outside the pool
             (5, [0, 1], [0, 1], [3], [-2]),
             (6, [0, 3], [0, 3], [29], None)]         # past the rotary tables
    for code, starts, bounds, first, table in cases:
        table = ints(table or [0, 1, 2])
        kp, _ = new_pool(4, Hk, D, torch.bfloat16, "paged_umma", dev, g)
        vp = kp.clone()
        before = kp.clone()
        rows = torch.randn(starts[-1], Hk, D, generator=g).to(torch.bfloat16).to(dev)
        status = torch.zeros(1, dtype=torch.int32, device=dev)
        q = rows.clone()
        ops.append_kv(rows, rows, kp, vp, "paged_umma", table, ints(bounds), ints(starts),
                      ints(first), q=q, cos=cos, sin=sin, status=status)
        assert int(status) == code
        changed = (kp != before).any(-1).any(1).sum().item()  # rows that were written
        ok = {30: 2, -1: 2, 29: 1, 3: 0}[first[0]]
        assert changed <= ok * D * 2
        if ok == 0:
            assert torch.equal(kp, before) and torch.equal(vp, before) and torch.equal(q, rows)
        if code != 6:
            out = torch.full_like(rows, 9.0)
            status.zero_()
            ops.read_kv(kp, vp, "paged_umma", table, ints(bounds), ints(starts), ints(first), out,
                        out.clone(), status=status)
            assert int(status) == code


def test_quantised_row_with_nan_or_infinity_reads_as_nan(cuda_device):
    from d2sd_b200 import ops
    dev, Hk, D = cuda_device, 1, 64
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    rows = torch.ones(4, Hk, D, dtype=torch.bfloat16, device=dev)
    rows[1, 0, 5], rows[2, 0, 63] = float("nan"), float("-inf")
    rows[3] *= 3e38
    kp = torch.zeros(1, Hk, 16, D, dtype=torch.uint8, device=dev).view(E4M3)
    vp = kp.clone()
    ks = torch.zeros(1, Hk, 16, dtype=torch.uint8, device=dev)
    vs = ks.clone()
    args = ("paged_umma", ints([0]), ints([0, 1]), ints([0, 4]), ints([0]))
    ops.append_kv(rows, rows, kp, vp, *args, k_scale=ks, v_scale=vs)
    ko, vo = torch.zeros_like(rows), torch.zeros_like(rows)
    ops.read_kv(kp, vp, *args, ko, vo, k_scale=ks, v_scale=vs)
    assert ko[1].isnan().all() and ko[2].isnan().all() and (ko[0] == 1).all()
    assert torch.equal(ko[3].double().cpu(), OP.e4m3_rows(rows[3].double().cpu())[0])


def test_refusals(cuda_device):
    import d2sd_b200 as d
    from d2sd_b200 import ops
    dev = cuda_device
    z = lambda *s, t=torch.bfloat16: torch.zeros(*s, dtype=t, device=dev)  # noqa: E731
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    kp, k = z(4, 2, 16, 64), z(3, 2, 64)
    one = (ints([0, 1, 2, 3]), ints([0, 4]), ints([0, 3]), ints([0]))

    def refused(err, *a, **kw):
        with pytest.raises(err):
            ops.append_kv(*a, **kw)
    refused(ValueError, k.float(), k.float(), kp, kp, "paged_umma", *one)      # cache type
    refused(ValueError, k, k, kp, kp, "nhd", *one)                             # not paged
    refused(ValueError, k[:, :1], k, kp, kp, "paged_umma", *one)               # heads
    refused(ValueError, k, k, kp, kp, "paged_umma", one[0].long(), *one[1:])   # int64 table
    refused(ValueError, k, k, kp, kp, "paged_umma", one[0], ints([0]), *one[2:])
    refused(ValueError, k, k, kp.view(E4M3) if False else z(4, 2, 16, 64, t=torch.uint8).view(E4M3),
            z(4, 2, 16, 64, t=torch.uint8).view(E4M3), "paged_umma", *one)     # no scales
    refused(ValueError, k, k, kp, kp, "paged_umma", *one, cos=z(9, 32, t=torch.float32))
    refused(NotImplementedError, k, k, kp, kp, "paged_umma", *one, cos=z(9, 20, t=torch.float32),
            sin=z(9, 20, t=torch.float32))                                     # rotary_dim 40
    refused(NotImplementedError, k[..., :32], k[..., :32], z(4, 2, 16, 32), z(4, 2, 16, 32),
            "paged_umma", *one)                                                # head_dim 32
    refused(ValueError, z(3, 2, 65)[..., 1:], k, kp, kp, "paged_umma", *one)   # alignment
    refused(ValueError, k.cpu(), k, kp, kp, "paged_umma", *one)
    with pytest.raises(ValueError):
        ops.read_kv(kp, kp, "paged_umma", *one, k.half(), k.half())
    # attention
    P = d.PagedAttentionPlan
    for bad in (dict(q_lens=[1], kv_lens=[1, 2]), dict(q_lens=[-1], kv_lens=[1]),
                dict(q_lens=[1, 1], kv_lens=[1, 1])):
        with pytest.raises(ValueError):
            P(bad["q_lens"], bad["kv_lens"], 4, 2, 64, dev)
    with pytest.raises(ValueError):
        P([1], [1], 5, 2, 64, dev)
    with pytest.raises(NotImplementedError):
        P([1], [1], 4, 2, 96, dev)
    with pytest.raises(NotImplementedError):
        P([1], [1], 4, 2, 64, dev, causal=False, window=3)
    with pytest.raises(NotImplementedError):
        P([1], [1], 129, 1, 64, dev)
    plan = P([3], [3], 4, 2, 64, dev)
    q, e8 = z(3, 4, 64), z(4, 2, 16, 64, t=torch.uint8).view(E4M3)
    for err, a, kw in [
            (ValueError, (q[:2], kp, kp, "paged_umma", one[0], plan), {}),
            (ValueError, (q.half(), kp, kp, "paged_umma", one[0], plan), {}),
            (NotImplementedError, (q.float(), kp.float(), kp.float(), "paged_hnd", one[0], plan), {}),
            (ValueError, (q, kp, kp, "paged_umma", one[0], plan), {"sinks": z(3, t=torch.float32)}),
            (ValueError, (q, kp[:, :1], kp[:, :1], "paged_hnd", one[0], plan), {}),
            (ValueError, (q, kp, kp, "paged_umma", one[0], plan), {"out": z(2, 4, 64)}),
            (ValueError, (q, kp, kp, "paged_umma", one[0][:0], plan), {}),     # a short page table
            (ValueError, (q, kp, kp, "paged_umma", one[0], plan), {"sm_scale": 0.0}),
            (NotImplementedError, (q.half(), e8, e8, "paged_umma", one[0], plan),
             {"k_scale": z(4, 2, 16, t=torch.uint8), "v_scale": z(4, 2, 16, t=torch.uint8)}),
            (NotImplementedError, (q, z(4, 2, 8, 64), z(4, 2, 8, 64), "paged_hnd", one[0], plan), {})]:
        with pytest.raises(err):
            d.paged_attention(*a, **kw)


# ---------------------------------------------------------------------------
# the operators together, through the caches
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("dtype,layout", [(torch.bfloat16, "umma"), (torch.bfloat16, "hnd"),
                                          (E4M3, "umma")])
def test_serving_steps_through_the_pool(cuda_device, dtype, layout):
    """Prompts in two chunks, then single tokens, of three sequences through one
    pool: each step appends (norm, rotary) and attends, against the same steps in
    float64 from the rows that the cache holds."""
    import d2sd_b200 as d
    dev = cuda_device
    L, Hq, Hk, D = 2, 8, 2, 128
    g = torch.Generator().manual_seed(77)
    pool = d.PagedKVPool(L, Hk, D, [400, 90, 300], dtype=dtype, device=dev, shuffle_seed=1,
                         layout=layout)
    cos, sin = d.rope_tables(512, D, 1e6, dev)
    w = [(1 + 0.2 * torch.randn(D, generator=g)).to(torch.bfloat16) for _ in range(2)]
    lens = [0, 0, 0]
    kept = [[[], []] for _ in range(3)]  # float64 k and v of each sequence, layer 1
    for new in ([150, 60, 9], [201, 0, 88], [1, 1, 1], [1, 1, 1]):
        n = sum(new)
        starts = torch.tensor([0] + list(np.cumsum(new)), dtype=torch.int32, device=dev)
        pool.set_lengths(lens)
        qkv = [torch.randn(n, Hq + 2 * Hk, D, generator=g).to(torch.bfloat16) for _ in range(L)]
        qs = []
        for l in range(L):
            x = qkv[l].to(dev)
            qs.append(pool.append(l, x[:, Hq:Hq + Hk], x[:, Hq + Hk:], starts, pool.lengths_dev,
                                  q=x[:, :Hq], q_weight=w[0].to(dev), k_weight=w[1].to(dev),
                                  cos=cos, sin=sin))
        pos = torch.cat([torch.arange(a, a + b) for a, b in zip(lens, new)])
        lens = [a + b for a, b in zip(lens, new)]
        pool.set_lengths(lens)
        plan = pool.plan(new, Hq)
        for l in range(L):
            ks, vs = pool.scales(l)
            out, lse = d.paged_attention(qs[l], pool.k[l], pool.v[l], pool.kv_layout,
                                         pool.page_table, plan, k_scale=ks, v_scale=vs)
        # layer 1: what append computes, then the attention of the rows the cache holds
        x = qkv[1].double()
        rot = lambda y, i: OP.norm_rotate(y, w[i], 1e-6, cos.cpu(), sin.cpu(), pos, False)  # noqa
        q64, k64 = rot(x[:, :Hq], 0), rot(x[:, Hq:Hq + Hk], 1)
        u = 2.0 ** -8
        got = qs[1].double().cpu()
        assert ((got - q64).abs() <= u * q64.abs() + 2.0 ** -17 * q64.abs().amax(-1, True) + 1e-30).all()
        at = 0
        for s, m in enumerate(new):
            kept[s][0].append(k64[at:at + m])
            kept[s][1].append(x[at:at + m, Hq + Hk:])
            at += m
        rows = [pool.gather_seq(1, s, lens[s]) for s in range(3)]
        for s in range(3):
            for i in range(2):
                want = torch.cat(kept[s][i])
                err = (rows[s][i].double().cpu() - want).abs()
                top = want.abs().amax(-1, keepdim=True)
                tol = ((2.0 ** -8 * want.abs() + 2.0 ** -17 * top) if dtype != E4M3 else
                       torch.maximum(want.abs() * 2.0 ** -4, top * 2 / 448 * 2.0 ** -10)
                       + 2.0 ** -17 * top)
                assert (err <= tol + 1e-30).all(), (s, i)
        c = dict(k_rows=[r[0].double().cpu() for r in rows], v_rows=[r[1].double().cpu() for r in rows])
        check_attention(out, lse, qs[1], c, new, D, torch.bfloat16)
    with pytest.raises(ValueError):
        pool.plan([1, 1], Hq)


@pytest.mark.parametrize("pooled", [False, True])
def test_commit_into_an_8bit_cache(cuda_device, pooled):
    import d2sd_b200 as d
    dev = cuda_device
    L, B, T, Hk, D = 3, 4, 16, 2, 64
    g = torch.Generator().manual_seed(12)
    S = 3 if pooled else 1
    lens = [37, 0, 16][:S]
    if pooled:
        cache = d.PagedKVPool(L, Hk, D, [80, 40, 33], dtype=E4M3, device=dev, shuffle_seed=3)
        cache.set_lengths(lens)
    else:
        cache = d.PagedKVCache(L, Hk, D, 80, dtype=E4M3, device=dev,
                               page_order=torch.randperm(5, generator=g))
        cache.length = 37
    old = []
    for s in range(S):
        x = torch.randn(lens[s], Hk, D, generator=g).to(torch.bfloat16)
        for l in range(L):
            if lens[s]:
                (cache.write_seq(l, s, x.to(dev), -x.to(dev)) if pooled else
                 cache.write(l, x.to(dev), -x.to(dev)))
        old.append(OP.e4m3_rows(x.double())[0])
    # the projections' token-major rows seen as [B, Hk, T, D]
    new = [torch.randn(2, S * B, T, Hk, D, generator=g).to(torch.bfloat16).to(dev) for _ in range(L)]
    nk, nv = [x[0].transpose(1, 2) for x in new], [x[1].transpose(1, 2) for x in new]
    res = torch.tensor([[5, 2], [16, 0], [1, 3]][:S], dtype=torch.int32, device=dev)
    if pooled:
        cache.commit_batch(nk, nv, res, B)
    else:
        cache.commit(nk, nv, res[0], advance_by=5)
        assert cache.length == 42
    for s in range(S):
        acc, b = res[s].tolist()
        for l in range(L):
            gk, gv = (cache.gather_seq(l, s, lens[s] + acc) if pooled else cache.gather(l))
            for i, (got, sign) in enumerate(((gk, 1), (gv, -1))):
                rows = new[l][i, s * B + b, :acc].double().cpu()
                want = torch.cat([sign * old[s], OP.e4m3_rows(rows)[0]])
                assert torch.equal(got.double().cpu(), want), (s, l, i)
    if not pooled:
        with pytest.raises(NotImplementedError):
            cache.commit(nk, nv, res[0], target_hidden=([torch.zeros(B, T, 64, device=dev)],
                                                        torch.zeros(T, 64, device=dev)))
        with pytest.raises(ValueError):
            d.PagedKVCache(1, Hk, D, 16, dtype=E4M3, device=dev, layout="hnd")
        with pytest.raises(ValueError):
            cache.write(0, torch.zeros(90, Hk, D, dtype=torch.bfloat16, device=dev),
                        torch.zeros(90, Hk, D, dtype=torch.bfloat16, device=dev))


def test_verify_forward_over_an_8bit_cache(cuda_device):
    """``cascade_verify_forward`` with an 8-bit PagedKVCache equals the same forward
    over a 16-bit cache of the rows that the 8-bit one stands for."""
    import d2sd_b200 as d
    from test_verification_gpu import tiny
    dev = cuda_device
    model = tiny("qwen3", dev)
    nl = len(model.model.layers)
    Hk, D = model.config.num_key_value_heads, model.model.layers[0].self_attn.head_dim
    g = torch.Generator().manual_seed(2)
    P, B, T = 137, 3, 8
    c8 = d.PagedKVCache(nl, Hk, D, 160, dtype=E4M3, device=dev)
    c16 = d.PagedKVCache(nl, Hk, D, 160, device=dev)
    for l in range(nl):
        k, v = (torch.randn(P, Hk, D, generator=g).to(torch.bfloat16).to(dev) for _ in range(2))
        c8.write(l, k, v)
        c16.write(l, *c8.gather(l, P))
    c8.length = c16.length = P
    ids = torch.randint(0, 512, (B, T), generator=g).to(dev)
    pos = torch.arange(P, P + T, device=dev).unsqueeze(0)
    a = d.cascade_verify_forward(model, ids, pos, c8)[0]
    b = d.cascade_verify_forward(model, ids, pos, c16)[0]
    assert torch.equal(a, b)


def test_page_bounds_behind_the_table_are_reported(cuda_device):
    """Bounds that give a request more pages than the table has: the positions behind
    its end are skipped with status 4, the others are written and read."""
    from d2sd_b200 import ops
    dev, Hk, D = cuda_device, 2, 128
    g = torch.Generator().manual_seed(31)
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    for dtype in (torch.bfloat16, E4M3):
        kp, ks = new_pool(6, Hk, D, dtype, "paged_umma", dev, g)
        vp, vs = kp.clone(), None if ks is None else ks.clone()
        rows = torch.randn(40, Hk, D, generator=g).to(torch.bfloat16).to(dev)
        status = torch.zeros(1, dtype=torch.int32, device=dev)
        args = ("paged_umma", ints([4, 2]), ints([0, 3]), ints([0, 40]), ints([0]))
        kw = dict(k_scale=ks, v_scale=vs, status=status)
        ops.append_kv(rows, rows, kp, vp, *args, **kw)
        assert int(status) == 4
        status.zero_()
        out = torch.full_like(rows, 9.0), torch.full_like(rows, 9.0)
        ops.read_kv(kp, vp, *args, *out, **kw)
        assert int(status) == 4
        want = rows[:32].double().cpu()
        if dtype == E4M3:
            want = OP.e4m3_rows(want)[0]
        for o in out:
            assert torch.equal(o[:32].double().cpu(), want) and (o[32:] == 9).all()


def test_commit_e4m3_skips_bad_positions_and_pages(cuda_device):
    from d2sd_b200 import ops
    dev, Hk, D, T = cuda_device, 2, 64, 8
    g = torch.Generator().manual_seed(33)
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    new = torch.randn(1, Hk, T, D, generator=g).to(torch.bfloat16).to(dev)
    # (status, page table, bounds, cached length, rows written)
    for code, table, bounds, length, written in ((4, [1], [0, 1], 12, 4), (4, [1], [0, 2], 12, 4),
                                                 (5, [1, 9], [0, 2], 12, 4), (0, [2, 0], [0, 2], 12, 8)):
        kp, ks = new_pool(3, Hk, D, E4M3, "paged_umma", dev, g)
        kp.view(torch.uint8).zero_()
        ks.zero_()
        vp, vs = kp.clone(), ks.clone()
        ptrs = torch.tensor([t.data_ptr() for t in (new, new, kp, vp, ks, vs)],
                            dtype=torch.int64, device=dev)
        status = torch.zeros(1, dtype=torch.int32, device=dev)
        ops.commit_kv_e4m3(ptrs, num_layers=1, num_requests=1, num_kv_heads=Hk, head_dim=D,
                           dtype=torch.bfloat16, block_len=T, new_strides=(0, *new.stride()[:3]),
                           cache_strides=kp.stride()[:2], num_pages=3, scale_strides=ks.stride()[:2],
                           page_table=ints(table), page_bounds=ints(bounds),
                           accept_results=ints([T, 0]), cache_lens=ints([length]), status=status)
        assert int(status) == code
        for s in (ks, vs):
            assert int((s != 0).sum()) == written * Hk


def test_commit_refuses_other_shapes(cuda_device):
    import d2sd_b200 as d
    cache = d.PagedKVCache(1, 2, 64, 64, dtype=E4M3, device=cuda_device)
    res = torch.tensor([1, 0], dtype=torch.int32, device=cuda_device)
    for shape in ((1, 3, 4, 64), (1, 2, 4, 128)):
        x = torch.zeros(shape, dtype=torch.bfloat16, device=cuda_device)
        with pytest.raises(ValueError):
            cache.commit([x], [x], res)
    x = torch.zeros(1, 2, 4, 64, dtype=torch.bfloat16, device=cuda_device)
    with pytest.raises(ValueError):
        cache.commit([x], [x[:, :, :3]], res)


def test_widened_pages_stay_within_a_bound(cuda_device, monkeypatch):
    """Above the bound of the scratch the pages are widened tile by tile instead."""
    import d2sd_b200 as d
    from d2sd_b200 import paged
    Hq, Hk, D, ql, kl = 16, 2, 128, [300], [1000]
    g = torch.Generator().manual_seed(35)
    c = make_cache(g, kl, Hk, D, E4M3, "paged_umma", cuda_device)
    q = torch.randn(300, Hq, D, generator=g).to(torch.bfloat16).to(cuda_device)
    for limit, widen in ((None, True), (63 * 16 * Hk * D * 4, True), (63 * 16 * Hk * D * 4 - 1, False)):
        if limit is not None:
            monkeypatch.setattr(paged, "_WIDE_BYTES", limit)
        plan = d.PagedAttentionPlan(ql, kl, Hq, Hk, D, cuda_device)
        assert plan.widen == widen and plan.wide_pages == 63
        out, lse = d.paged_attention(q, c["k"], c["v"], "paged_umma", c["table"], plan,
                                     k_scale=c["ks"], v_scale=c["vs"])
        check_attention(out, lse, q, c, ql, D, torch.bfloat16)


def test_window_larger_than_any_length(cuda_device):
    import d2sd_b200 as d
    Hq, Hk, D, ql, kl = 8, 2, 64, [3, 40, 2], [3, 100, 0]
    g = torch.Generator().manual_seed(37)
    c = make_cache(g, kl, Hk, D, torch.float16, "paged_hnd", cuda_device)
    q = torch.randn(sum(ql), Hq, D, generator=g).half().to(cuda_device)
    for window in (2 ** 31 - 1, 2 ** 31 + 5, 2 ** 32 + 5):
        plan = d.PagedAttentionPlan(ql, kl, Hq, Hk, D, cuda_device, window=window,
                                    page_offsets=c["bounds"])
        out, lse = d.paged_attention(q, c["k"], c["v"], "paged_hnd", c["table"], plan)
        check_attention(out, lse, q, c, ql, D, torch.float16)


@pytest.mark.parametrize("D,dtype,layout", [(128, torch.bfloat16, "paged_umma"), (64, torch.float16, "paged_hnd"),
                                            (64, E4M3, "paged_umma"), (128, E4M3, "paged_umma")])
@pytest.mark.parametrize("R", [1, 9, 18])
def test_attention_in_clusters(cuda_device, D, dtype, layout, R):
    """Plans of clusters of 8, 4 and 2 CTAs: ragged lengths, a request without a key,
    windows and sinks; and the same plan through an update to one without clusters."""
    import d2sd_b200 as d
    Hq, Hk = 16, 8
    qt = torch.bfloat16 if dtype == E4M3 else dtype
    g = torch.Generator().manual_seed(41 + R)
    ql = [1 + i % 8 for i in range(R)]
    kl = [400] + [(137 * i) % 401 for i in range(1, R)]
    if R > 1:
        kl[3], kl[4] = 0, ql[4] - 2
    c = make_cache(g, kl, Hk, D, dtype, layout, cuda_device, garbage=True)
    q = torch.randn(sum(ql), Hq, D, generator=g).to(qt).to(cuda_device)
    sinks = torch.randn(Hq, generator=g).to(cuda_device)
    kw = dict(cache_dtype=dtype, page_offsets=c["bounds"])
    for window, s in ((None, None), (150, sinks)):
        plan = d.PagedAttentionPlan(ql, kl, Hq, Hk, D, cuda_device, window=window, **kw)
        if window is None:
            assert plan.sections[7] == {1: 8, 9: 4, 18: 2}[R] and plan.sections[3] == 0
        run = lambda: d.paged_attention(q, c["k"], c["v"], layout, c["table"], plan, k_scale=c["ks"],  # noqa: E731
                                        v_scale=c["vs"], sinks=s)
        out, lse = run()
        check_attention(out, lse, q, c, ql, D, qt, window=window, sinks=None if s is None else s.cpu())
        again, _ = run()
        assert torch.equal(out, again)
        plan.update([1] * R, [min(n, 100) for n in kl], c["bounds"])
        assert plan.sections[7] <= 1 or plan.sections[3] > 0
        plan.update(ql, kl, c["bounds"])
        again, _ = run()
        assert torch.equal(out, again)


@pytest.mark.parametrize("Hq,Hk,D,ql,kl,window", [
    (32, 8, 128, [1, 2, 0, 1, 2, 1], [1, 2, 40, 17, 3001, 1500], None),
    (64, 8, 64, [1] * 5, [0, 15, 16, 700, 2100], None),
    (6, 2, 128, [2, 1, 2], [333, 90, 1], 50),
    (8, 8, 64, [8, 3, 5], [1100, 2, 129], 300),
    (8, 1, 128, [1], [60000], None),
    (32, 8, 128, [1] * 80, [37 * i for i in range(80)], None),
])
def test_eight_bit_units_of_up_to_eight_rows(cuda_device, Hq, Hk, D, ql, kl, window):
    import d2sd_b200 as d
    g = torch.Generator().manual_seed(51)
    c = make_cache(g, kl, Hk, D, E4M3, "paged_umma", cuda_device, garbage=True)
    n = sum(ql)
    # rows of very different sizes: each is scaled by a power of two of its own
    q = torch.randn(n, Hq, D, generator=g) * 2.0 ** torch.randint(-9, 3, (n, Hq, 1), generator=g)
    q = q.to(torch.bfloat16).to(cuda_device)
    sinks = torch.randn(Hq, generator=g).to(cuda_device)
    plan = d.PagedAttentionPlan(ql, kl, Hq, Hk, D, cuda_device, window=window, page_offsets=c["bounds"],
                                cache_dtype=E4M3)
    assert plan.sections[19] == 0 and plan.sections[9] == 0  # the form of few rows alone
    for s in (None, sinks):
        out, lse = d.paged_attention(q, c["k"], c["v"], "paged_umma", c["table"], plan, k_scale=c["ks"],
                                     v_scale=c["vs"], sinks=s)
        check_attention(out, lse, q, c, ql, D, torch.bfloat16, window=window, sinks=None if s is None else s.cpu())
    assert int(plan.status) == 0


@pytest.mark.parametrize("Hq,Hk,D,dtype,layout,ql,kl,window", [
    (32, 8, 128, torch.bfloat16, "paged_umma", [1, 2, 0, 1, 2, 1], [1, 2, 40, 17, 3001, 1500], None),
    (10, 2, 64, torch.float16, "paged_umma", [1] * 5, [0, 15, 16, 700, 2100], None),
    (6, 2, 128, torch.float16, "paged_hnd", [2, 1, 2], [333, 90, 1], 50),
    (8, 8, 64, torch.bfloat16, "paged_nhd", [8, 3, 5], [1100, 2, 129], 300),
    (32, 8, 64, torch.float16, "paged_hnd", [1] * 80, [37 * i for i in range(80)], None),
])
def test_units_of_up_to_eight_rows(cuda_device, Hq, Hk, D, dtype, layout, ql, kl, window):
    import d2sd_b200 as d
    g = torch.Generator().manual_seed(53)
    c = make_cache(g, kl, Hk, D, dtype, layout, cuda_device, garbage=True)
    q = torch.randn(sum(ql), Hq, D, generator=g).to(dtype).to(cuda_device)
    sinks = torch.randn(Hq, generator=g).to(cuda_device)
    plan = d.PagedAttentionPlan(ql, kl, Hq, Hk, D, cuda_device, window=window, page_offsets=c["bounds"])
    assert plan.sections[19] == 0 and plan.sections[9] == 0  # the form of few rows alone
    for s in (None, sinks):
        out, lse = d.paged_attention(q, c["k"], c["v"], layout, c["table"], plan, sinks=s)
        check_attention(out, lse, q, c, ql, D, dtype, window=window, sinks=None if s is None else s.cpu())
    assert int(plan.status) == 0


@pytest.mark.parametrize("interleaved", [False, True])
def test_quantised_keys_are_the_nearest(cuda_device, interleaved):
    """8-bit keys after norm and rotation are the e4m3 values nearest to the 64-bit ones.
    fp32 is off by at most 4 last places of the rotation's larger operand (inverse root,
    product by it, two products, their sum), and values within 16 of their own of a border
    are decided in 64 bits; so only a value under a quarter of its operands may differ."""
    from d2sd_b200 import ops, rope_tables
    dev, n, Hk, D = cuda_device, 8192, 8, 128
    g = torch.Generator(device=dev).manual_seed(61)
    k = (torch.randn(n, Hk, D, generator=g, device=dev) * 1.7).to(torch.bfloat16)
    w = (1 + 0.2 * torch.randn(D, generator=g, device=dev)).to(torch.bfloat16)
    cos, sin = rope_tables(n, D, 1e6, dev)
    kp = torch.zeros(n // 16, Hk, 16, D, dtype=torch.uint8, device=dev).view(E4M3)
    vp, ks = kp.clone(), torch.zeros(n // 16, Hk, 16, dtype=torch.uint8, device=dev)
    vs = ks.clone()
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    args = ("paged_umma", torch.arange(n // 16, dtype=torch.int32, device=dev), ints([0, n // 16]),
            ints([0, n]), ints([0]))
    ops.append_kv(k, k, kp, vp, *args, k_scale=ks, v_scale=vs, k_weight=w, cos=cos, sin=sin,
                  interleaved=interleaved)
    got, v = torch.empty_like(k), torch.empty_like(k)
    ops.read_kv(kp, vp, *args, got, v, k_scale=ks, v_scale=vs)
    x = k.double()
    y = x / (x.square().mean(-1, keepdim=True) + 1e-6).sqrt() * w.double()
    c, s = cos.double()[:, None], sin.double()[:, None]
    a, b = (y[..., 0::2], y[..., 1::2]) if interleaved else (y[..., :D // 2], y[..., D // 2:])
    pair = (a * c - b * s, b * c + a * s), (a * c).abs() + (b * s).abs(), (b * c).abs() + (a * s).abs()
    join = (lambda p: torch.stack(p, -1).flatten(-2)) if interleaved else (lambda p: torch.cat(p, -1))
    f, size = join(pair[0]), join(pair[1:])
    unit = torch.exp2(ks.view(n // 16, Hk, 16).transpose(1, 2).reshape(n, Hk, 1).double() - 127)
    # the border test in 64 bits: |f - got| against the distance to the neighbours
    step = torch.exp2(torch.floor(torch.log2((f.abs() / unit).clamp(min=2.0 ** -6))) - 3) * unit
    off = (got.double() - f).abs() > step / 2
    assert int((off & (f.abs() >= size / 4)).sum()) == 0
    assert int(off.sum()) < 64  # of 8.4 million


@pytest.mark.parametrize("dtype", [torch.bfloat16, E4M3])
@pytest.mark.parametrize("longest", [1, 2, 5])
def test_captured_decode_steps(cuda_device, dtype, longest):
    """Reserved plans that say how many new tokens a request has at most: the captured call
    of up to 8, 16 and 32 query rows replays, and longer requests are refused."""
    import d2sd_b200 as d
    Hq, Hk, D, R = 32, 8, 64, 3
    g = torch.Generator().manual_seed(71)
    full = [1100, 300, 2500]
    c = make_cache(g, full, Hk, D, dtype, "paged_umma", cuda_device)
    q = torch.randn(R * longest, Hq, D, generator=g).to(torch.bfloat16).to(cuda_device)
    plan = d.PagedAttentionPlan([1] * R, [9] * R, Hq, Hk, D, cuda_device, page_offsets=c["bounds"],
                                cache_dtype=dtype, reserve=(R, R * longest, longest))
    out, lse = torch.zeros_like(q), torch.zeros(len(q), Hq, device=cuda_device)
    call = lambda: d.paged_attention(q, c["k"], c["v"], "paged_umma", c["table"], plan, k_scale=c["ks"],  # noqa: E731
                                     v_scale=c["vs"], out=out, lse=lse)
    call()
    s = torch.cuda.Stream(cuda_device)
    s.wait_stream(torch.cuda.current_stream(cuda_device))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(s), torch.cuda.graph(graph, stream=s):
        call()
    torch.cuda.current_stream(cuda_device).wait_stream(s)
    for ql, kl in (([1] * R, [9] * R), ([longest, 1, longest], [1100, 16, 2500]), ([0, longest, 0], [7, 300, 9]),
                   ([longest] * R, [longest - 1, longest, 2000])):
        plan.update(ql, kl, c["bounds"])
        graph.replay()
        torch.cuda.synchronize(cuda_device)
        cut = dict(c, k_rows=[x[:n] for x, n in zip(c["k_rows"], kl)],
                   v_rows=[x[:n] for x, n in zip(c["v_rows"], kl)])
        check_attention(out, lse, q, cut, ql, D, torch.bfloat16)
    with pytest.raises(ValueError):
        plan.update([longest + 1, 0, 0], [50] * 3, c["bounds"])
    assert int(plan.status) == 0
    del graph
