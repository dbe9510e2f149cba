"""Calls of the paged-cache operators next to their limits: values, sinks and sizes that
ordinary batches do not have. Tolerances as in test_paged_gpu.py."""
import pytest
import torch

from oracle import paged as OP
from test_paged_gpu import E4M3, check_attention, make_cache

pytestmark = pytest.mark.gpu


# ---------------------------------------------------------------------------
# a NaN code of e4m3 under a finite scale
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("n,widen", [(1, False), (12, False), (40, False), (300, True)])
@pytest.mark.parametrize("code", [0x7f, 0xff])
def test_nan_code_of_e4m3_is_nan_in_every_form(cuda_device, D, n, widen, code):
    """A pool may hold e4m3's NaN in a row with an ordinary scale byte (torch's cast
    makes it). Position 0, which every row sees: a NaN in the value row is a NaN in that
    column of every row, one in the key row makes the rows of its head NaN."""
    import d2sd_b200 as d
    Hq, Hk, kl = 8, 2, 400
    g = torch.Generator().manual_seed(90 + n)
    c = make_cache(g, [kl], Hk, D, E4M3, "paged_umma", cuda_device)
    q = torch.randn(n, Hq, D, generator=g).to(torch.bfloat16).to(cuda_device)
    plan = d.PagedAttentionPlan([n], [kl], Hq, Hk, D, cuda_device, cache_dtype=E4M3)
    assert plan.widen == widen
    col = D - 3
    run = lambda c: d.paged_attention(q, c["k"], c["v"], "paged_umma", c["table"], plan,  # noqa: E731
                                      k_scale=c["ks"], v_scale=c["vs"])[0]

    def planted(pool):  # position 0 of kv head 1
        x = pool.clone()
        page = int(c["table"][0])
        x.view(torch.uint8)[page, 1].flatten()[OP.page_index("paged_umma", D, 1)[0, col]] = code
        return x
    base = run(c)
    out = run(dict(c, v=planted(c["v"])))
    nan = torch.zeros_like(out, dtype=torch.bool)
    nan[:, Hq // 2:, col] = True
    assert torch.equal(out.isnan(), nan)
    assert torch.equal(out[~nan], base[~nan])
    out = run(dict(c, k=planted(c["k"])))
    assert out[:, Hq // 2:].isnan().all() and torch.equal(out[:, :Hq // 2], base[:, :Hq // 2])


# ---------------------------------------------------------------------------
# one key far above all others
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("type,layout", [("f16", "paged_umma"), ("f16", "paged_hnd"), ("bf16", "paged_umma"),
                                         ("e4m3", "paged_umma")])
@pytest.mark.parametrize("n,kl", [(1, 2000), (4, 2000), (1, 20000), (160, 2000), (40, 9000)])
@pytest.mark.parametrize("at", [0, 900])
def test_weights_far_below_the_largest(cuda_device, type, layout, n, kl, at):
    """A key 16.26 nats (23.5 binades) above all others, whose value row has one column:
    the other columns are the sum of the others' weights, each of the same relative
    error as any."""
    import d2sd_b200 as d
    Hq, Hk, D = 8, 2, 64
    dt = torch.float16 if type == "f16" else torch.bfloat16
    g = torch.Generator().manual_seed(95)
    c = make_cache(g, [kl], Hk, D, E4M3 if type == "e4m3" else dt, layout, cuda_device)
    k, v = torch.zeros(kl, Hk, D), torch.ones(kl, Hk, D)
    k[at, :, 0] = 1.0
    v[at] = 0.0
    v[at, :, 5] = 1.0
    q = torch.zeros(n, Hq, D)
    q[:, :, 0] = 16.25
    page_rows = {"k": k, "v": v}
    for x, rows in page_rows.items():  # as plain rows or core matrices, scales of one
        blocks = torch.zeros(-(-kl // 16) * 16, Hk, D)
        blocks[:kl] = rows
        blocks = blocks.view(-1, 16, Hk, D).transpose(1, 2)
        store = E4M3 if type == "e4m3" else dt
        val, byte = OP.e4m3_rows(blocks.double())
        if type == "e4m3":
            blocks = (val / 2.0 ** (byte.double() - 127)[..., None]).float()
            c[x + "s"][c["table"].long()] = byte.to(cuda_device)
        flat = torch.empty(len(blocks), Hk, 16 * D)
        flat[..., OP.page_index(layout, D, store.itemsize).flatten()] = blocks.flatten(2)
        new = flat.view(-1, Hk, 16, D).to(store).to(cuda_device)
        bits = torch.uint8 if type == "e4m3" else store
        c[x].view(bits)[c["table"].long()] = new.view(bits)
    c["k_rows"], c["v_rows"] = [k.double()], [v.double()]
    q = q.to(dt).to(cuda_device)
    plan = d.PagedAttentionPlan([n], [kl], Hq, Hk, D, cuda_device, cache_dtype=c["k"].dtype)
    out, lse = d.paged_attention(q, c["k"], c["v"], layout, c["table"], plan, sm_scale=1.0,
                                 k_scale=c["ks"], v_scale=c["vs"])
    check_attention(out, lse, q, c, [n], D, dt, scale=1.0)


# ---------------------------------------------------------------------------
# sinks of -inf
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("Hq,Hk,D,store,ql,kl,kind", [
    (8, 2, 128, "bf16", [1, 3, 2], [5, 1, 0], "whole"),
    (16, 8, 64, "bf16", [8], [400], "cluster"), (16, 8, 64, "e4m3", [8, 5], [400, 3], "cluster"),
    (8, 1, 128, "bf16", [2], [20000], "join"), (8, 8, 64, "bf16", [300, 20], [130, 0], "tiles"),
    (4, 1, 128, "e4m3", [700], [690], "tiles"),
])
def test_sinks_of_minus_infinity(cuda_device, Hq, Hk, D, store, ql, kl, kind):
    """A head with a sink of -inf has none: nothing is taken from its rows, and a row
    without a key still gets 0."""
    import d2sd_b200 as d
    g = torch.Generator().manual_seed(99)
    dt = E4M3 if store == "e4m3" else torch.bfloat16
    c = make_cache(g, kl, Hk, D, dt, "paged_umma", cuda_device, garbage=True)
    q = torch.randn(sum(ql), Hq, D, generator=g).to(torch.bfloat16).to(cuda_device)
    sinks = torch.randn(Hq, generator=g).to(cuda_device)
    sinks[::2] = float("-inf")
    plan = d.PagedAttentionPlan(ql, kl, Hq, Hk, D, cuda_device, page_offsets=c["bounds"], cache_dtype=dt)
    s = plan.sections
    assert {"whole": s[1] > 0 and s[7] <= 1, "cluster": s[7] > 1 and s[3] == 0, "join": s[3] > 0,
            "tiles": s[9] > 0}[kind]
    for mode in ("exact", "reference"):
        out, lse = d.paged_attention(q, c["k"], c["v"], "paged_umma", c["table"], plan, k_scale=c["ks"],
                                     v_scale=c["vs"], sinks=sinks, sink_mode=mode)
        check_attention(out, lse, q, c, ql, D, torch.bfloat16, sinks=sinks.cpu(), sink_mode=mode)


@pytest.mark.parametrize("n", [1, 4])
def test_weights_of_large_8bit_values(cuda_device, n):
    """Values near the top of fp32's range, whose exponent the weights' reference holds:
    one key 17 binades above the others keeps them."""
    import d2sd_b200 as d
    Hq, Hk, D, kl = 8, 2, 64, 300
    g = torch.Generator().manual_seed(97)
    c = make_cache(g, [kl], Hk, D, E4M3, "paged_umma", cuda_device)
    one = torch.zeros(16, D, dtype=torch.float64)
    one[:, 0] = 1.0
    for x, rows, byte in (("k", one, 127), ("v", one * 0 + 256, 127 + 112)):
        flat = torch.empty(16 * D, dtype=torch.uint8)
        flat[OP.page_index("paged_umma", D, 1).flatten()] = rows.float().to(E4M3).view(torch.uint8).flatten()
        c[x].view(torch.uint8).flatten(2)[:] = flat.to(cuda_device)
        c[x + "s"].fill_(byte)
    # scores by the key's scale: 2^(byte - 127) q_0; position 20 above all others
    c["ks"].fill_(100)
    c["ks"][c["table"][1].long(), :, 4] = 127
    pages = c["table"].long().cpu()
    c["k_rows"] = [OP.cached_rows(c["k"], "paged_umma", pages, kl, c["ks"])]
    c["v_rows"] = [OP.cached_rows(c["v"], "paged_umma", pages, kl, c["vs"])]
    q = torch.zeros(n, Hq, D)
    q[..., 0] = 12.0
    q = q.to(torch.bfloat16).to(cuda_device)
    plan = d.PagedAttentionPlan([n], [kl], Hq, Hk, D, cuda_device, cache_dtype=E4M3)
    out, lse = d.paged_attention(q, c["k"], c["v"], "paged_umma", c["table"], plan, sm_scale=1.0,
                                 k_scale=c["ks"], v_scale=c["vs"])
    check_attention(out, lse, q, c, [n], D, torch.bfloat16, scale=1.0)


# ---------------------------------------------------------------------------
# 8-bit keys next to a border
# ---------------------------------------------------------------------------
def quantise(k, w, cos, sin, interleaved, eps=1e-6):
    """append_kv of k as one request's rows from position 0: (what they read as, scale bytes)."""
    from d2sd_b200 import ops
    n, Hk, D = k.shape
    dev = k.device
    pages = -(-n // 16)
    kp = torch.zeros(pages, Hk, 16, D, dtype=torch.uint8, device=dev).view(E4M3)
    vp, ks = kp.clone(), torch.zeros(pages, Hk, 16, dtype=torch.uint8, device=dev)
    vs = ks.clone()
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    args = ("paged_umma", torch.arange(pages, dtype=torch.int32, device=dev), ints([0, pages]), ints([0, n]),
            ints([0]))
    ops.append_kv(k, k, kp, vp, *args, k_scale=ks, v_scale=vs, k_weight=w, cos=cos, sin=sin,
                  interleaved=interleaved, eps=eps)
    got, v = torch.empty_like(k), torch.empty_like(k)
    ops.read_kv(kp, vp, *args, got, v, k_scale=ks, v_scale=vs)
    return got, ks.transpose(1, 2).reshape(-1, Hk)[:n]


def keys_64(k, w, cos, sin, interleaved, eps=1e-6):
    """Norm and rotation of rows 0.. in 64 bits."""
    y = k.double()
    if w is not None:
        y = y / (y.square().mean(-1, keepdim=True) + eps).sqrt() * w.double()
    if cos is None:
        return y
    c, s = cos[:len(k)].double()[:, None], sin[:len(k)].double()[:, None]
    h = cos.shape[1]
    a, b = (y[..., 0:2 * h:2], y[..., 1:2 * h:2]) if interleaved else (y[..., :h], y[..., h:2 * h])
    p = a * c - b * s, b * c + a * s
    turned = torch.stack(p, -1).flatten(-2) if interleaved else torch.cat(p, -1)
    return torch.cat([turned, y[..., 2 * h:]], -1)


def check_nearest(got, byte, f):
    """The scale is that of the definition and every value the nearest e4m3 one: off by at
    most half of the step at the exact value (2^-9 of the scale at the least; 2^-40 of it
    for what 64 bits themselves round)."""
    top = f.abs().amax(-1)
    unit = torch.exp2(byte.double() - 127)
    assert bool((top <= 448 * unit).all())
    assert bool(((top > 224 * unit) | (byte == 1)).all())
    step = torch.exp2(torch.floor(torch.log2((f.abs() / unit[..., None]).clamp(min=2.0 ** -6))) - 3) * unit[..., None]
    off = (got.double() - f).abs() > step / 2 * (1 + 2.0 ** -40)
    assert int(off.sum()) == 0, int(off.sum())


def cancelling_tables(n, half, device):
    """cos = 1 and sin = 1 - d, d of 2^-16 to 2^-8: equal pairs nearly cancel."""
    g = torch.Generator(device=device).manual_seed(109)
    d = 2.0 ** -(8 + 8 * torch.rand(n, half, generator=g, device=device))
    return torch.ones(n, half, device=device), 1 - d


@pytest.mark.parametrize("type", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D,rot,interleaved,norm", [(128, 128, False, True), (128, 128, True, True),
                                                    (64, 32, False, True), (128, 96, True, False),
                                                    (64, 0, False, True)])
@pytest.mark.parametrize("spread", [0, 8, "cancel"])
def test_quantised_keys_are_the_nearest_ones(cuda_device, type, D, rot, interleaved, norm, spread):
    """8.4 million values: none rounded past a border, however small it is beside its row
    (spread: columns of different sizes, down to 2^-spread) or its rotation's operands."""
    from d2sd_b200 import rope_tables
    dev, n, Hk = cuda_device, 8192, 1024 // D
    g = torch.Generator(device=dev).manual_seed(101)
    k = torch.randn(n, Hk, D, generator=g, device=dev) * 1.7
    if spread == "cancel":
        k = 1.5 + torch.rand(n, Hk, 1, generator=g, device=dev).expand(n, Hk, D)
    elif spread:
        k *= 2.0 ** -(spread * torch.rand(D, generator=g, device=dev)).round()
    k = k.to(type)
    w = (1 + 0.2 * torch.randn(D, generator=g, device=dev)).to(type) if norm else None
    cos, sin = rope_tables(n, rot, 1e6, dev) if rot else (None, None)
    if spread == "cancel" and rot:
        w = torch.full_like(w, 1.25) if norm else None
        cos, sin = cancelling_tables(n, rot // 2, dev)
    got, byte = quantise(k, w, cos, sin, interleaved)
    f = keys_64(k, w, cos, sin, interleaved)
    if type == torch.float16:  # read into fp16, whose own step is coarser under 2^-14
        got = torch.where(f.abs() >= 2.0 ** -13, got.double(), f)
    check_nearest(got, byte, f)


def test_scale_of_a_row_next_to_its_border(cuda_device):
    """Rows whose largest value is 448 * 2^e to within a last place of fp32: each has the
    scale of its exact value. The norm's eps is what puts it there."""
    dev, D = cuda_device, 64
    g = torch.Generator(device=dev).manual_seed(103)
    w = torch.ones(D, dtype=torch.bfloat16, device=dev)
    for i in range(200):
        k = torch.randn(1, 1, D, generator=g, device=dev).to(torch.bfloat16)
        x = k.double().flatten()
        top, mean = float(x.abs().max()), float(x.square().mean())
        target = 1.75 * 2.0 ** -2  # the border under most rows' normalised maximum
        assert (top / target) ** 2 > mean
        eps = float(torch.tensor((top / target) ** 2 - mean, dtype=torch.float32))
        got, byte = quantise(k, w, None, None, False, eps=eps)
        check_nearest(got, byte, keys_64(k, w, None, None, False, eps=eps))


@pytest.mark.parametrize("D", [64, 128])
def test_a_tokens_keys_do_not_depend_on_its_batch(cuda_device, D):
    """The same token beside 4096 others (even rows; one table row for all) has the same
    bytes every time, values next to a border included."""
    dev, n, Hk = cuda_device, 8192, 8
    g = torch.Generator(device=dev).manual_seed(107)
    w = torch.full((D,), 1.25, dtype=torch.bfloat16, device=dev)
    for i in range(12):
        cos, sin = (t[i:i + 1].expand(n, -1).contiguous() for t in cancelling_tables(12, D // 2, dev))
        k = torch.randn(n, Hk, D, generator=g, device=dev)
        k[::2] = 1.5 + torch.rand(1, Hk, 1, generator=g, device=dev)
        got, byte = quantise(k.to(torch.bfloat16), w, cos, sin, False)
        assert bool((got[::2] == got[0]).all()) and bool((byte[::2] == byte[0]).all()), i


# ---------------------------------------------------------------------------
# lengths above a sequence's pages
# ---------------------------------------------------------------------------
def test_pool_refuses_lengths_above_capacity(cuda_device):
    """Positions behind a sequence's capacity would be the next sequence's rows."""
    import d2sd_b200 as d
    pool = d.PagedKVPool(1, 2, 64, [40, 100, 33], device=cuda_device)
    for bad in ([41, 0, 0], [0, 101, 0], [0, 0, 34], [-1, 0, 0], [1, 1]):
        with pytest.raises(ValueError):
            pool.set_lengths(bad)
    assert pool.lengths == [0, 0, 0]
    pool.set_lengths([40, 100, 33])
    plan = pool.plan([1, 2, 3], 4)
    with pytest.raises(ValueError):
        plan.update([1, 2, 3], [41, 100, 33], pool.page_offsets_host)
    with pytest.raises(ValueError):
        pool.plan([1, 2, 3], 4, reserve=(3, 6)).update([1, 2, 3], [40, 100, 48], pool.page_offsets_host)
    plan.update([1, 2, 3], [40, 99, 33], pool.page_offsets_host)
    pool.lengths[0] += 1
    with pytest.raises(ValueError):
        pool.plan([1, 2, 3], 4)


@pytest.mark.parametrize("layout,page_size", [("paged_umma", 16), ("paged_hnd", 32)])
def test_page_bounds_limit_every_request(cuda_device, layout, page_size):
    """Plans with page bounds: a request longer than its own pages is refused, though the
    page table goes on."""
    import d2sd_b200 as d
    Hq, Hk, D = 4, 2, 64
    g = torch.Generator().manual_seed(111)
    kl = [3 * page_size, 2 * page_size]
    c = make_cache(g, kl, Hk, D, torch.bfloat16, layout, cuda_device, page_size=page_size)
    q = torch.randn(2, Hq, D, generator=g).to(torch.bfloat16).to(cuda_device)
    run = lambda plan: d.paged_attention(q, c["k"], c["v"], layout, c["table"], plan)  # noqa: E731
    plan = d.PagedAttentionPlan([1, 1], kl, Hq, Hk, D, cuda_device, page_offsets=c["bounds"])
    out, lse = run(plan)
    check_attention(out, lse, q, c, [1, 1], D, torch.bfloat16)
    plan.update([1, 1], [3 * page_size + 1, 5], c["bounds"])
    with pytest.raises(ValueError):
        run(plan)
    plan.update([1, 1], kl, c["bounds"])
    again, _ = run(plan)
    assert torch.equal(out, again)


def test_updates_fit_the_page_table_of_a_captured_call(cuda_device):
    """A replay reads the page table that its call was captured with: an update to
    lengths that go on behind it is refused, and the plan stays as it was."""
    import d2sd_b200 as d
    Hq, Hk, D = 8, 2, 64
    g = torch.Generator().manual_seed(113)
    c = make_cache(g, [200, 90], Hk, D, torch.bfloat16, "paged_umma", cuda_device)
    q = torch.randn(2, Hq, D, generator=g).to(torch.bfloat16).to(cuda_device)
    plan = d.PagedAttentionPlan([1, 1], [20, 30], Hq, Hk, D, cuda_device, page_offsets=c["bounds"][:2],
                                reserve=(2, 2, 1))
    out, lse = torch.zeros_like(q), torch.zeros(2, Hq, device=cuda_device)
    call = lambda: d.paged_attention(q, c["k"], c["v"], "paged_umma", c["table"], plan, out=out, lse=lse)  # noqa
    call()
    plan.update([1, 1], [200, 90 + 17], c["bounds"][:2])  # a longer table may come with the next call
    plan.update([1, 1], [20, 30], c["bounds"][:2])
    s = torch.cuda.Stream(cuda_device)
    s.wait_stream(torch.cuda.current_stream(cuda_device))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(s), torch.cuda.graph(graph, stream=s):
        call()
    torch.cuda.current_stream(cuda_device).wait_stream(s)
    for kl in ([200, 90], [200, 90 + 17], [5, 90]):
        if kl[1] > 96:
            with pytest.raises(ValueError):
                plan.update([1, 1], kl, c["bounds"][:2])
            kl = [200, 90]
        else:
            plan.update([1, 1], kl, c["bounds"][:2])
        out.zero_()
        graph.replay()
        torch.cuda.synchronize(cuda_device)
        cut = dict(c, k_rows=[x[:n] for x, n in zip(c["k_rows"], kl)],
                   v_rows=[x[:n] for x, n in zip(c["v_rows"], kl)])
        check_attention(out, lse, q, cut, [1, 1], D, torch.bfloat16)
    del graph


# ---------------------------------------------------------------------------
# rows that are not there, through the caches
# ---------------------------------------------------------------------------
def test_8bit_rows_behind_the_cache_are_refused(cuda_device):
    """gather and gather_seq of more rows than there are raise, instead of returning
    memory that nothing wrote; a negative start is refused."""
    import d2sd_b200 as d
    cache = d.PagedKVCache(1, 2, 64, 32, dtype=E4M3, device=cuda_device)
    pool = d.PagedKVPool(1, 2, 64, [20, 40], dtype=E4M3, device=cuda_device)
    x = torch.ones(16, 2, 64, dtype=torch.bfloat16, device=cuda_device)
    for call in (lambda: cache.gather(0, 33), lambda: cache.gather(0, -1), lambda: pool.gather_seq(0, 0, 21),
                 lambda: pool.gather_seq(0, 1, 41), lambda: pool.gather(0, 81),
                 lambda: cache.write(0, x, x, start=-1), lambda: cache.write(0, x, x, start=17)):
        with pytest.raises(ValueError):
            call()
    for got, n in ((cache.gather(0, 32), 32), (pool.gather_seq(0, 0, 20), 20), (pool.gather(0, 80), 80)):
        assert got[0].shape == (n, 2, 64) and not got[0].any() and not got[1].any()
    assert int(cache.status) == 0 and int(pool.status) == 0


def test_gather_of_a_pool_is_the_same_in_both_types(cuda_device):
    """The pool's gather goes over the whole page table, whatever the cache's type."""
    import d2sd_b200 as d
    g = torch.Generator().manual_seed(117)
    pools = [d.PagedKVPool(1, 2, 64, [20, 40, 5], dtype=t, device=cuda_device, shuffle_seed=2)
             for t in (torch.bfloat16, E4M3)]
    for s, n in enumerate([20, 40, 5]):
        x = torch.randint(-8, 9, (n, 2, 64), generator=g).to(torch.bfloat16).to(cuda_device)
        for p in pools:
            p.write_seq(0, s, x, -x)
    for n in (7, 20, 33, 96):
        a, b = (p.gather(0, n) for p in pools)
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_status_of_the_caches(cuda_device):
    """A commit past a sequence's pages, an append past them and a bad page are reported
    by the cache's own status; a tensor that is passed is used instead."""
    import d2sd_b200 as d
    dev = cuda_device
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    new = torch.ones(2, 2, 8, 64, dtype=torch.bfloat16, device=dev)
    pool = d.PagedKVPool(1, 2, 64, [16, 40], dtype=E4M3, device=dev)
    pool.set_lengths([10, 20])
    pool.commit_batch([new], [new], ints([[6, 0], [8, 0]]), 1)
    assert int(pool.status) == 0
    pool.commit_batch([new], [new], ints([[7, 0], [8, 0]]), 1)  # position 16 of a page of 16
    assert int(pool.status) == 4
    for dtype in (torch.bfloat16, E4M3):
        pool = d.PagedKVPool(1, 2, 64, [16, 40], dtype=dtype, device=dev)
        rows = torch.ones(5, 2, 64, dtype=torch.bfloat16, device=dev)
        starts, first = ints([0, 3, 5]), ints([14, 0])
        own = ints([0])
        pool.append(0, rows, rows, starts, first, status=own)
        assert int(own) == 4 and int(pool.status) == 0
        pool.append(0, rows, rows, starts, first)
        assert int(pool.status) == 4
        pool.status.zero_()
        out = torch.zeros_like(rows)
        pool.read(0, starts, first, out, out.clone())
        assert int(pool.status) == 4
        pool.status.zero_()
        pool.page_table[2] = 99
        pool.append(0, rows, rows, starts, ints([3, 10]))
        assert int(pool.status) == 0
        pool.append(0, rows, rows, starts, ints([3, 16]))
        assert int(pool.status) == 5
    cache = d.PagedKVCache(1, 2, 64, 32, dtype=E4M3, device=dev, page_order=torch.tensor([0, 1]))
    cache.page_table[1] = -1
    cache.commit([new[:1]], [new[:1]], ints([8, 0]), cache_len=12)
    assert int(cache.status) == 5


# ---------------------------------------------------------------------------
# arguments of the wrong size or type
# ---------------------------------------------------------------------------
def test_sizes_of_device_arguments(cuda_device):
    """What a kernel reads or writes by the number of requests is checked against it."""
    import d2sd_b200 as d
    from d2sd_b200 import ops
    dev = cuda_device
    ints = lambda x, t=torch.int32: torch.tensor(x, dtype=t, device=dev)  # noqa: E731
    pool = d.PagedKVPool(1, 2, 64, [40, 40], dtype=E4M3, device=dev)
    new = torch.zeros(2, 2, 8, 64, dtype=torch.bfloat16, device=dev)
    for res in (ints([1, 0]), ints([[1, 0], [1, 0]], torch.int64)):
        with pytest.raises(ValueError):
            pool.commit_batch([new], [new], res, 1)
    pool.commit_batch([new], [new], ints([[1, 0]] * 3), 1)  # of a verifier of more requests
    pool.lengths_dev = ints([0])
    with pytest.raises(ValueError):
        pool.commit_batch([new], [new], ints([[1, 0], [1, 0]]), 1)
    kw = dict(num_layers=1, num_requests=1, num_kv_heads=2, head_dim=64, dtype=torch.bfloat16, block_len=8,
              new_strides=(0, *new.stride()[:3]), cache_strides=pool.k[0].stride()[:2], num_pages=6,
              scale_strides=pool.k_scale[0].stride()[:2], page_table=pool.page_table, page_bounds=ints([0, 3]),
              accept_results=ints([0, 0]), cache_lens=ints([0]))
    ptrs = [t.data_ptr() for t in (new, new, pool.k, pool.v, pool.k_scale, pool.v_scale)]
    ops.commit_kv_e4m3(ints(ptrs, torch.int64), **kw)
    for bad in (ints(ptrs[:4], torch.int64), torch.zeros(6, dtype=torch.float64, device=dev)):
        with pytest.raises(ValueError):
            ops.commit_kv_e4m3(bad, **kw)
    rows = torch.zeros(2, 2, 64, dtype=torch.bfloat16, device=dev)
    args = (ints([0, 2]), ints([0]))
    cache = d.PagedKVCache(1, 2, 64, 32, device=dev)
    for status in (ints([0], torch.uint8), ints([0], torch.int64), ints([])):
        with pytest.raises(ValueError):
            cache.append(0, rows, rows, *args, status=status)
        with pytest.raises(ValueError):
            cache.read(0, *args, rows, rows.clone(), status=status)
        with pytest.raises(ValueError):
            ops.commit_kv_e4m3(ints(ptrs, torch.int64), status=status, **kw)


# ---------------------------------------------------------------------------
# verify blocks right behind the launch that writes them
# ---------------------------------------------------------------------------
def test_verify_block_behind_append_and_read(cuda_device):
    """q rotated in place by append, k and v read out of the cache, and at once the block's
    attention (no prefix; a dense one; an empty paged one): as with a wait between."""
    import d2sd_b200 as d
    from d2sd_b200 import CascadeGraphRunner, single_prefill_with_kv_cache
    dev, Hq, Hk, D, n, T = cuda_device, 32, 8, 128, 4096, 16
    g = torch.Generator(device=dev).manual_seed(121)
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    cache = d.PagedKVCache(1, Hk, D, n, device=dev)
    cos, sin = d.rope_tables(n, D, 1e6, dev)
    starts, first = ints([0, n]), ints([0])
    runner = CascadeGraphRunner(T, Hq, Hk, D, torch.bfloat16, dev, D ** -0.5, True)
    plan = d.CascadePlan([d.Request(2 * T, 0, 0, 0)], Hq, Hk, D, dev)
    dense = (torch.randn(2, T, Hq, D, generator=g, device=dev).to(torch.bfloat16),
             torch.randn(2, T, Hq, generator=g, device=dev))

    def step(qkv, form, wait):
        q, kr, vr = qkv[:, :Hq].clone(), torch.zeros(n, Hk, D, dtype=torch.bfloat16, device=dev), None
        vr, out = kr.clone(), tuple(t.clone() for t in dense)
        torch.cuda.synchronize(dev)
        cache.append(0, qkv[:, Hq:Hq + Hk], qkv[:, Hq + Hk:], starts, first, q=q, cos=cos, sin=sin)
        cache.read(0, starts, first, kr, vr)
        if form == "append":  # q last: rotated once more, in place
            cache.append(0, kr, vr, starts, first, q=q, cos=cos, sin=sin)
        if wait:
            torch.cuda.synchronize(dev)
        b = lambda t: t[-2 * T:].view(2, T, *t.shape[1:])  # noqa: E731
        if form == "runner":
            runner.run(b(q), b(kr), b(vr), *out)
            return out
        if form == "cascade":
            return d.cascade_attention(b(q), b(kr), b(vr), cache.k[0], cache.v[0], cache.kv_layout, 0,
                                       page_table=cache.page_table, plan=plan)
        return single_prefill_with_kv_cache(q[-T:], kr[-T:], vr[-T:], causal=True, return_lse=True)

    runner.run(*(torch.zeros(2, T, h, D, dtype=torch.bfloat16, device=dev) for h in (Hq, Hk, Hk)),
               *(t.clone() for t in dense))
    for i in range(6):
        qkv = torch.randn(n, Hq + 2 * Hk, D, generator=g, device=dev).to(torch.bfloat16)
        for form in ("append", "read", "runner", "cascade"):
            for a, b in zip(step(qkv, form, False), step(qkv, form, True)):
                assert torch.equal(a, b), (i, form)


# ---------------------------------------------------------------------------
# the log-sum-exp of few keys
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("type", ["bf16", "f16", "e4m3"])
@pytest.mark.parametrize("kl", [1, 2, 40, 300])
@pytest.mark.parametrize("n", [1, 70])
def test_lse_of_small_scores(cuda_device, type, kl, n):
    """Scores near zero: the log-sum-exp is as exact as its own size, whatever the values'
    exponents are (8-bit rows from 2^-17 to 1 here). The score's error, 2^-22 for the
    exponentials, (kl + 8) 2^-24 for their sum, and two steps of the result at its size
    or 1."""
    import d2sd_b200 as d
    Hq, Hk, D = 8, 2, 64
    dt = torch.float16 if type == "f16" else torch.bfloat16
    g = torch.Generator().manual_seed(131)
    c = make_cache(g, [kl], Hk, D, E4M3 if type == "e4m3" else dt, "paged_umma", cuda_device)
    if type == "e4m3":
        byte = torch.randint(102, 120, c["vs"].shape, generator=g).to(torch.uint8)
        c["vs"].copy_(byte)
    q = torch.randn(n, Hq, D, generator=g).to(dt).to(cuda_device)
    plan = d.PagedAttentionPlan([n], [kl], Hq, Hk, D, cuda_device, cache_dtype=c["k"].dtype)
    out, lse = d.paged_attention(q, c["k"], c["v"], "paged_umma", c["table"], plan, sm_scale=1e-3,
                                 k_scale=c["ks"], v_scale=c["vs"])
    v = OP.cached_rows(c["v"], "paged_umma", c["table"].cpu().long(), kl, None if type != "e4m3" else c["vs"])
    _, want, _, big = OP.attention(q.double().cpu(), c["k_rows"][0], v, scale=1e-3)
    got = lse.double().cpu()
    empty = want == float("-inf")
    assert torch.equal(got == float("-inf"), empty)
    tol = ((D + 4) * 2.0 ** -24 * big + 2.0 ** -22 + (min(kl, 300) + 8) * 2.0 ** -24) * 1.4427 \
        + 2 * 2.0 ** -23 * want.abs().clamp(min=1.0)
    assert ((got - want).abs() <= tol)[~empty].all(), float((got - want).abs()[~empty].max())


def test_reserves_of_no_size_are_refused(cuda_device):
    import d2sd_b200 as d
    for reserve in ((0, 4), (1, 0), (1, 4, 0), (1,), (1, 4, 1, 1), (-1, 4)):
        with pytest.raises(ValueError):
            d.PagedAttentionPlan([], [], 4, 2, 64, cuda_device, reserve=reserve)
    plan = d.PagedAttentionPlan([], [], 4, 2, 64, cuda_device, reserve=(1, 4, 4))
    plan.update([4], [9])
    with pytest.raises(ValueError):
        plan.update([5], [9])
