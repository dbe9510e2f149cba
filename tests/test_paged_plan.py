"""The host-side plan of the paged attention (CPU only): every (row, visible key
tile) of every request in exactly one item, spans in order, the slots and the list
of rows to join, and the balance over the CTAs."""
import numpy as np
import pytest


@pytest.fixture(scope="module")
def lib():
    from d2sd_b200 import build
    build.build()
    from d2sd_b200 import _lib
    return _lib.load()


def make(lib, q, kv, off, Hq, Hk, causal, window, ctas, eight_bit=0):
    from d2sd_b200._lib import check
    q, kv, off = (np.ascontiguousarray(x, dtype=np.int32) for x in (q, kv, off))
    cap = lib.d2sd_paged_plan_capacity(q.ctypes.data, len(q), Hq, Hk, ctas)
    plan, used, sec = np.zeros(cap, np.int32), np.zeros(1, np.int64), np.zeros(20, np.int32)
    check(lib.d2sd_paged_plan(q.ctypes.data, kv.ctypes.data, off.ctypes.data, len(q), Hq, Hk, causal,
                              window, eight_bit, ctas, plan.ctypes.data, cap, used.ctypes.data,
                              sec.ctypes.data), "plan")
    return plan[:int(used[0])], sec


@pytest.mark.parametrize("eight_bit", [0, 1])
@pytest.mark.parametrize("q,kv,Hq,Hk,causal,window,ctas", [
    ([1] * 64, list(range(512, 8193, 120))[:64], 32, 8, 1, 0, 148),
    ([1], [1000], 32, 8, 1, 0, 148),
    ([1], [1], 8, 8, 1, 0, 148),
    ([5, 0, 16, 1], [5, 40, 300, 0], 10, 2, 1, 0, 7),
    ([900, 3], [900, 5000], 32, 8, 1, 0, 148),
    ([900, 3], [1900, 5000], 64, 8, 1, 128, 148),
    ([4, 9], [70, 0], 16, 4, 0, 0, 148),
    ([2048], [32768], 32, 8, 1, 0, 148),
    ([100], [40], 4, 2, 1, 0, 5),
    ([3] * 300, [77] * 300, 8, 1, 1, 0, 3),
])
def test_plan_covers_every_tile_once(lib, eight_bit, q, kv, Hq, Hk, causal, window, ctas):
    off = np.cumsum([0] + [-(-n // 16) for n in kv])[:-1]
    plan, sec = make(lib, q, kv, off, Hq, Hk, causal, window, ctas, eight_bit)
    G = Hq // Hk
    starts = np.cumsum([0] + list(q))
    seen = {}
    for s in range(2):
        nct, nit, nslots, njoin, oc, oi, oj, most_parts = sec[8 * s:8 * s + 8]
        assert list(plan[5 + 8 * s:13 + 8 * s]) == list(sec[8 * s:8 * s + 8])
        if nit == 0:
            continue
        q_tile = 16 if s == 0 else 128 // G * G
        cta = plan[oc:oc + nct + 1]
        most = 4 * ctas if s == 0 else ctas
        assert nct <= most and cta[0] == 0 and cta[-1] == nit and (np.diff(cta) >= 0).all()
        assert nslots <= 2 * most and oi % 4 == 0
        items = plan[oi:oi + 16 * nit].reshape(-1, 16)
        slots, split = set(), {}
        for it in items:
            r, h, tok0, row0, nrows, k0, k1, pos0, win, po, kvl, slot, parts, tokb, *_ = it
            assert tok0 == starts[r] and po == off[r] and kvl == kv[r] and win == window
            assert 0 < nrows <= (q_tile if s == 0 else 2 * q_tile)
            assert row0 + nrows <= q[r] * G and k0 % 16 == 0 and k1 <= kv[r]
            assert tokb == row0 // G and (s == 0 or (row0 % G == 0 and nrows % G == 0))
            unit = seen.setdefault((r, h, row0), [nrows, []])
            unit[1].append((k0, k1))
            if parts == 1:
                assert slot == -1
            else:
                first = split.setdefault((r, h, row0), (slot, parts, nrows, tok0))[0]
                assert slot == first + len(unit[1]) - 1 and slot not in slots  # spans in slot order
                slots.add(slot)
        assert slots == set(range(nslots))
        assert most_parts == max([x[1] for x in split.values()], default=1)
        # join list: every row of every split unit once, with its slot
        joined = {}
        for j in plan[oj:oj + 8 * njoin].reshape(-1, 8):
            slot, step, parts, srow, n, row0, tok0, head = j
            assert 0 < n <= (4, 8)[s] and step == (1, 2)[s] and srow + n <= q_tile
            for x in range(n):
                key = (tok0, head, row0 + x)
                assert key not in joined
                joined[key] = (slot, parts, srow + x)
        want = {}
        for (r, h, row0), (first, parts, nrows, tok0) in split.items():
            for x in range(nrows):
                tile, rest = divmod(x, q_tile)
                want[tok0, h, row0 + x] = (first * (1, 2)[s] + tile, parts, rest)
        assert joined == want
        # balance: the largest CTA within the mean and two items' fixed costs
        extra = 1 if s == 0 else 4
        cost = [sum((-(-(i[6] - i[5]) // 128) + extra) * (2 if s == 1 and i[4] > q_tile else 1)
                    for i in items[a:b]) for a, b in zip(cta, cta[1:])]
        assert max(cost) <= sum(cost) / nct + 2 * (extra + 2) * 2
    for r in range(len(q)):
        rows = q[r] * G
        for h in range(Hk):
            units = sorted((k[2], v) for k, v in seen.items() if k[:2] == (r, h))
            at = 0
            for row0, (n, spans) in units:
                assert row0 == at
                at += n
                pos0 = kv[r] - q[r]
                hi, lo = kv[r], 0
                if causal:
                    hi = max(0, min(kv[r], pos0 + (row0 + n - 1) // G + 1))
                    lo = max(0, pos0 + row0 // G + 1 - window) if window else 0
                lo = min(lo // 16 * 16, hi)
                assert spans[0][0] == lo and spans[-1][1] == hi
                for a, b in zip(spans, spans[1:]):
                    assert a[1] == b[0] and b[1] > b[0] and (a[1] - a[0]) % 128 == 0
            assert at == rows


def test_plan_refusals(lib):
    with pytest.raises(ValueError):
        make(lib, [1], [-1], [0], 4, 2, 1, 0, 8)
    with pytest.raises(ValueError):
        make(lib, [1], [1], [-1], 4, 2, 1, 0, 8)
    with pytest.raises(ValueError):
        make(lib, [1], [1], [0], 4, 2, 1, -3, 8)
    with pytest.raises(NotImplementedError):
        make(lib, [1], [1], [0], 4, 2, 0, 16, 8)
    with pytest.raises(NotImplementedError):
        make(lib, [1], [1 << 30], [0], 4, 2, 1, 0, 8)
    with pytest.raises(NotImplementedError):
        make(lib, [1], [1], [0], 129, 1, 1, 0, 8)
    import ctypes
    n = np.ones(1, np.int32)
    buf, used, sec = np.zeros(4, np.int32), np.zeros(1, np.int64), np.zeros(20, np.int32)
    rc = lib.d2sd_paged_plan(n.ctypes.data, n.ctypes.data, ctypes.c_void_p(np.zeros(1, np.int32).ctypes.data),
                             1, 4, 2, 1, 0, 0, 8, buf.ctypes.data, 4, used.ctypes.data, sec.ctypes.data)
    assert rc == 3 and "small" in lib.d2sd_last_error().decode()
    assert lib.d2sd_paged_plan_capacity(n.ctypes.data, 1, 5, 2, 8) == -1
    assert lib.d2sd_paged_workspace_bytes(148, 96) == -1


def test_empty_batches(lib):
    plan, sec = make(lib, [], [], [], 4, 2, 1, 0, 8)
    assert sec[1] == 0 and sec[9] == 0
    plan, sec = make(lib, [0, 0], [7, 0], [0, 1], 4, 2, 1, 0, 8)
    assert sec[1] == 0 and sec[9] == 0


def test_e4m3_oracle_against_the_type():
    """The oracle's 8-bit rows against torch's own rounding to float8_e4m3fn."""
    import torch
    from oracle import paged as OP
    g = torch.Generator().manual_seed(0)
    x = torch.randn(500, 64, generator=g) * 2.0 ** torch.randint(-130, 20, (500, 1), generator=g).float()
    x[0] = 0
    vals, byte = OP.e4m3_rows(x.double())
    e = byte.double() - 127
    top = x.double().abs().amax(-1)
    assert (top <= 448 * 2.0 ** e).all() and ((top > 448 * 2.0 ** (e - 1)) | (e == -126)).all()
    y = x.double() / (2.0 ** e)[:, None]
    assert torch.equal(y.float().to(torch.float8_e4m3fn).double() * (2.0 ** e)[:, None], vals)


def test_window_above_every_position(lib):
    """The largest window an int32 holds is the plan of no position left out, rows
    without a key (fewer cached positions than new tokens) included."""
    args = ([1, 40, 7], [5, 900, 2], [0, 1, 58], 8, 2, 1)
    plan, _ = make(lib, *args, 2 ** 31 - 1, 16)
    free, _ = make(lib, *args, 1 << 30, 16)
    assert np.array_equal(plan, free)


@pytest.mark.parametrize("q,kv,Hq,Hk,window,ctas", [
    ([4000], [4000], 32, 8, 0, 148),            # a prompt: row tiles of rising cost
    ([700, 301, 999], [700, 4000, 999], 64, 8, 128, 148),
    ([1] * 200, [50 + 7 * i for i in range(200)], 8, 8, 0, 100),
])
def test_many_units_stay_whole(lib, q, kv, Hq, Hk, window, ctas):
    """Where whole units balance, none is cut, and no CTA has more than its share and
    the cost of cutting."""
    off = np.cumsum([0] + [-(-n // 16) for n in kv])[:-1]
    plan, sec = make(lib, q, kv, off, Hq, Hk, 1, window, ctas)
    s = 0 if sec[1] else 1
    n, items, slots, joins, oc, oi, _, parts = sec[8 * s:8 * s + 8]
    extra = 1 if s == 0 else 4
    assert n == (4 * ctas if s == 0 else ctas) and slots == 0 and joins == 0 and parts == 1
    it = plan[oi:oi + 16 * items].reshape(items, 16)
    pair = 2 * (128 // (Hq // Hk)) * (Hq // Hk)
    weight = np.where((it[:, 4] > pair // 2) & (s == 1), 2, 1)
    cost = (-(-(it[:, 6] - it[:, 5]) // 128) + extra) * weight
    load = [cost[plan[oc + c]:plan[oc + c + 1]].sum() for c in range(n)]
    assert plan[oc] == 0 and plan[oc + n] == items and min(load) > 0
    share = cost.sum() // n
    assert max(load) <= share + max(2 * extra * weight.max(), share // 64)


def test_packed_calls_are_checked(lib):
    """d2sd_call: an unknown entry and a wrong number of words."""
    words = b"\0" * 8 * 64
    for entry, n in ((-1, 44), (3, 44), (0, 43), (1, 44), (2, 64)):
        assert lib.d2sd_call(entry, words, n) == 1 and "d2sd_call" in lib.d2sd_last_error().decode()
    assert lib.d2sd_call(0, None, 45) == 1


@pytest.mark.parametrize("q,kv,Hq,Hk,window", [([1], [1000], 32, 8, 0), ([4], [130], 32, 8, 0),
                                               ([1, 0, 3, 2], [2001, 7, 0, 129], 8, 2, 300),
                                               ([1], [4096], 64, 8, 0), ([3], [4000], 40, 8, 17 + 512)])
def test_plan_of_clusters(lib, q, kv, Hq, Hk, window):
    """Few units: eight consecutive CTAs of one item each for every unit, their spans of
    whole pages in order and without a gap, and nothing to join."""
    off = np.cumsum([0] + [-(-n // 16) for n in kv])[:-1]
    plan, sec = make(lib, q, kv, off, Hq, Hk, 1, window, 148, 2)
    n, items, slots, joins, oc, oi, _, parts = sec[:8]
    assert parts in (4, 8) and slots == 0 and joins == 0 and n == items and n % parts == 0 and n <= 592
    assert list(plan[oc:oc + n + 1]) == list(range(n + 1))
    it = plan[oi:oi + 16 * items].reshape(-1, parts, 16)
    G, seen = Hq // Hk, set()
    for unit in it:
        r, head, row0, rows = unit[0, 0], unit[0, 1], unit[0, 3], unit[0, 4]
        assert (unit[:, [0, 1, 2, 3, 4, 7, 8, 9, 10]] == unit[0, [0, 1, 2, 3, 4, 7, 8, 9, 10]]).all()
        assert (unit[1:, 5] == unit[:-1, 6]).all() and (unit[:, 5] <= unit[:, 6]).all()
        last = kv[r] - q[r] + (row0 + rows - 1) // G
        lo = max(0, kv[r] - q[r] + row0 // G + 1 - window) if window else 0
        assert unit[0, 5] <= lo or last < 0
        assert unit[-1, 6] == max(last + 1, 0)
        inner = unit[:, 5][unit[:, 5] < unit[:, 6]]
        assert (inner % 16 == 0).all()
        seen |= {(r, head, x) for x in range(row0, row0 + rows)}
    assert seen == {(r, h, x) for r in range(len(q)) for h in range(Hk) for x in range(q[r] * G)}
    # longer prefixes and many units are cut over all CTAs
    assert make(lib, [1], [9000], [0], Hq, Hk, 1, 0, 148, 2)[1][3] > 0
