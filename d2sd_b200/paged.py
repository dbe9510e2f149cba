"""The target's own attention over its paged cache.

``paged_attention`` runs a ragged batch of new tokens -- prompts in chunks, single
tokens, drafted blocks taken as plain sequences -- against the cache that
``ops.append_kv`` has just written them into: causal, with an optional sliding
window and attention sinks, over 16-bit or e4m3 pages. ``PagedAttentionPlan`` is
its plan/run split, as ``CascadePlan`` is kernel (a)'s: built on the host from the
lengths once per step, used by every layer.
"""
from __future__ import annotations

import math

import numpy as np
import torch

from . import _lib, ops
from ._lib import check, load

_WIDE_BYTES = 4 << 30  # scratch of widened pages: a million positions of 8 heads of 128
_SINKS = {"reference": _lib.SINK_REFERENCE, "exact": _lib.SINK_EXACT}


class PagedAttentionPlan:
    """Work plan and workspace of ``paged_attention`` for one ragged batch.

    q_lens / kv_lens: new tokens of each request and its cached positions, the new
    ones included (the new tokens are the last of them). page_offsets: each
    request's first entry in the page table (default: one request from entry 0, or
    ``PagedKVPool.page_offsets_host``). With an entry more (page bounds, ascending) a
    request with more cached positions than its pages hold is refused by the call; with
    capacities, the positions that each request has room for, by the plan and ``update``
    (``PagedKVPool.plan`` gives them). Without either, such a request reads on in the
    page table.
    window: a row sees only the last ``window`` positions up to its own. cache_dtype:
    float8_e4m3fn chooses the kernels for an 8-bit cache (any plan works with any).

    The plan owns the workspace of its calls: two calls that overlap on the GPU
    need a plan each. ``update`` re-plans in place, on the current stream. With
    ``reserve=(requests, tokens)`` the device buffers have room for that many, the
    tensors of a call must hold that many tokens, and the launch does not depend on
    the lengths: a captured ``paged_attention`` replays with the updated ones (of a
    plan without a reserve it must not be replayed after an update). A third number,
    the most new tokens of one request, saves the launches that only longer ones need
    (1 for a decode step; up to 16 query rows per kv head). Planning takes 15 us of host
    time for one request, 50 for 64 and 1 ms for 1024; the plan's way to the GPU waits for
    what is queued on the stream. Plans with a reserve do not widen 8-bit pages ahead
    (2048 tokens over 32k positions 1320 us instead of 920).
    """

    def __init__(self, q_lens, kv_lens, num_qo_heads: int, num_kv_heads: int, head_dim: int,
                 device: torch.device | str, *, causal: bool = True, window: int | None = None,
                 page_offsets=None, capacities=None, cache_dtype: torch.dtype | None = None,
                 reserve: tuple[int, ...] | None = None):
        device = torch.device(device)
        if device.type != "cuda":
            raise ValueError("PagedAttentionPlan needs a CUDA device")
        if window is not None and window <= 0:
            raise ValueError("window must be positive")
        self.num_qo_heads, self.num_kv_heads, self.head_dim = num_qo_heads, num_kv_heads, head_dim
        self.causal, self.window = causal, window
        self.capacities = None if capacities is None else np.asarray(capacities, dtype=np.int64)
        self._captured = set()  # (page size, entries of the page table) of captured calls
        self.eight_bit = int(cache_dtype == torch.float8_e4m3fn)
        self.num_ctas = ops.num_sms(device)
        self.reserve = reserve
        self.fixed_grid = 0
        if reserve is not None:
            if len(reserve) not in (2, 3) or min(reserve) <= 0:
                raise ValueError("reserve is (requests, tokens) or (requests, tokens, most of a "
                                 "request), all positive")
            self.longest = reserve[2] if len(reserve) > 2 else reserve[1]
            rows = self.longest * num_qo_heads // num_kv_heads
            self.fixed_grid = _lib.GRID_FIXED
            if rows <= (32 if self.eight_bit else 16):
                self.fixed_grid |= _lib.GRID_FEW_ROWS
            if rows <= 8:
                self.fixed_grid |= _lib.GRID_EIGHT_ROWS
        host, sections, tokens = self._plan(q_lens, kv_lens, page_offsets)
        need = len(host)
        if reserve is not None:
            # most units: one long request and the others of one token each
            lens = np.ones(reserve[0], dtype=np.int32)
            lens[0] = reserve[1]
            need = load().d2sd_paged_plan_capacity(lens.ctypes.data, len(lens), num_qo_heads,
                                                   num_kv_heads, self.num_ctas)
        with torch.cuda.device(device):
            self.plan = torch.zeros(need, dtype=torch.int32, device=device)
            self.device = self.plan.device
            nbytes = load().d2sd_paged_workspace_bytes(self.num_ctas, head_dim)
            if nbytes < 0:
                raise NotImplementedError("paged attention: head_dim must be 64 or 128")
            self.workspace = torch.empty(nbytes, dtype=torch.uint8, device=device)
            self.status = torch.zeros(1, dtype=torch.int32, device=device)
            self._f32 = torch.empty(0, dtype=torch.float32, device=device)  # new_empty: less host time
            self._set(host, sections, tokens)
            torch.cuda.current_stream(device).synchronize()  # usable on any stream from here

    def _plan(self, q_lens, kv_lens, page_offsets):
        q = np.ascontiguousarray(q_lens, dtype=np.int32)
        kv = np.ascontiguousarray(kv_lens, dtype=np.int32)
        R = len(q)
        if q.ndim != 1 or kv.shape != q.shape:
            raise ValueError("q_lens and kv_lens must be lists of the same length")
        if page_offsets is None:
            if R > 1:
                raise ValueError("page_offsets are required for several requests")
            page_offsets = [0] * R
        if self.reserve is not None and (R > self.reserve[0] or int(q.sum()) > self.reserve[1]
                                         or int(q.max(initial=0)) > self.longest):
            raise ValueError(f"the batch is larger than the plan's reserve {self.reserve}")
        bounds = np.ascontiguousarray(page_offsets, dtype=np.int32)
        off = bounds[:R]
        if len(off) != R:
            raise ValueError("page_offsets must have an entry for each request")
        if self.capacities is not None and (len(self.capacities) < R
                                            or (kv > self.capacities[:R]).any()):
            raise ValueError("kv_lens are above the requests' capacities")
        ends = bounds[1:R + 1] if len(bounds) > R and (bounds[1:R + 1] >= off).all() else None
        requests = (kv, off, ends)
        for page_size, entries in self._captured:
            if self._pages(requests, page_size) > entries:
                raise ValueError("the page table of a captured call is too short for these lengths")
        lib = load()
        cap = lib.d2sd_paged_plan_capacity(q.ctypes.data, R, self.num_qo_heads, self.num_kv_heads,
                                           self.num_ctas)
        if cap < 0:
            raise ValueError("invalid plan sizes")
        plan = np.empty(cap, dtype=np.int32)
        used = np.zeros(1, dtype=np.int64)
        sections = np.zeros(20, dtype=np.int32)
        check(lib.d2sd_paged_plan(q.ctypes.data, kv.ctypes.data, off.ctypes.data, R,
                                  self.num_qo_heads, self.num_kv_heads, 1 if self.causal else 0,
                                  min(self.window or 0, 1 << 30), self.eight_bit + (0 if self.fixed_grid else 2),
                                  self.num_ctas, plan.ctypes.data, cap,
                                  used.ctypes.data, sections.ctypes.data), "d2sd_paged_plan")
        self._requests, self._entries = requests, {}
        return plan[:int(used[0])], sections, int(q.sum())

    @staticmethod
    def _pages(requests, page_size: int) -> int:
        kv, off, ends = requests
        last = off.astype(np.int64) + -(-kv.astype(np.int64) // page_size)
        if ends is not None and (last > ends).any():
            r = int((last > ends).argmax())
            raise ValueError(f"request {r} has {kv[r]} cached positions, more than its pages hold")
        return int(last.max(initial=0))

    def entries(self, page_size: int) -> int:
        """Entries that a page table must have for pages of this size."""
        n = self._entries.get(page_size)
        if n is None:
            n = self._entries[page_size] = self._pages(self._requests, page_size)
        return n

    def _set(self, host, sections, tokens):
        self.plan[:len(host)].copy_(torch.from_numpy(host))
        self.host_plan, self.sections, self.tokens = host, sections, tokens
        # an 8-bit cache is widened first where its keys are gone over three times or
        # more (32 query heads over 16k tokens: 128 new tokens 76 us either way, 256
        # 106 against 117, 2048 over 32k 1060 against 1330), not where the launch has
        # to fit any batch or the scratch would be a cache of its own
        self.wide_pages = int(sections[18] - sections[17])
        wide_bytes = self.wide_pages * self.num_kv_heads * 16 * self.head_dim * 4
        self.widen = int(sections[16]) >= 3 and not self.fixed_grid and wide_bytes <= _WIDE_BYTES
        # what every call passes on
        self._args = (self.plan.data_ptr(), sections.ctypes.data, self.num_ctas,
                      self.fixed_grid, self.workspace.data_ptr(),
                      self.workspace.numel())

    def update(self, q_lens, kv_lens, page_offsets=None) -> None:
        """Plan another batch into the same device buffers, on the current stream."""
        new = self._plan(q_lens, kv_lens, page_offsets)
        if len(new[0]) > self.plan.numel() and not self.fixed_grid:
            self.plan = torch.empty(2 * len(new[0]), dtype=torch.int32, device=self.device)
        self._set(*new)


def paged_attention(q: torch.Tensor, k_pool: torch.Tensor, v_pool: torch.Tensor, kv_layout: str,
                    page_table: torch.Tensor, plan: PagedAttentionPlan, *,
                    sm_scale: float | None = None, k_scale: torch.Tensor | None = None,
                    v_scale: torch.Tensor | None = None, sinks: torch.Tensor | None = None,
                    sink_mode: str = "exact", out: torch.Tensor | None = None,
                    lse: torch.Tensor | None = None):
    """q [tokens, Hq, D] (bf16 or fp16; bf16 with an e4m3 cache), the planned
    requests' new tokens one after another; pools per ``kv_layout`` ("paged_umma",
    "paged_hnd" or "paged_nhd") with their int32 ``page_table``; k_scale / v_scale
    uint8 [pages, Hk, 16] for an e4m3 cache. sinks fp32 [Hq]: out times
    sigmoid(lse - sink) (``sink_mode`` as in ``cascade_attention``).

    Returns (out [tokens, Hq, D], lse [tokens, Hq] fp32, base 2), written into
    ``out`` / ``lse`` when given; rows behind the plan's tokens are left alone. A
    row that sees no key has out 0 and lse -inf. Prompt chunks over an e4m3 cache
    take scratch of 4 * Hk * D bytes for each of their positions (up to 4 GiB; above
    it the pages are widened tile by tile). Cache slots past a request's last
    position may hold anything. A NaN or an infinity in the value of a position that
    some row of a tile sees may reach rows of that tile that do not see it."""
    dev = q.get_device()
    ops._same_device(dev, plan.status, k_pool, v_pool, page_table, k_scale, v_scale, sinks, out, lse)
    Hq, Hk, D = plan.num_qo_heads, plan.num_kv_heads, plan.head_dim
    dtype, n = q.dtype, q.shape[0]
    tokens = plan.reserve[1] if plan.reserve else plan.tokens
    if n < tokens:
        raise ValueError(f"q must hold the plan's {tokens} tokens")
    pool, heads, dim = ops._pool_args(k_pool, v_pool, kv_layout, k_scale, v_scale)
    if heads != Hk or dim != D:
        raise ValueError("the pools and the plan differ in kv heads or head_dim")
    if k_pool.dtype != dtype and k_pool.dtype != torch.float8_e4m3fn:
        raise ValueError(f"a {k_pool.dtype} cache does not take {dtype} queries")
    if dtype == torch.float32:
        raise NotImplementedError("paged attention takes bf16 or fp16 queries")
    if sinks is not None and (sinks.dtype != torch.float32 or not sinks.is_contiguous()
                              or sinks.numel() != Hq):
        raise ValueError("sinks must be a contiguous fp32 tensor [num_qo_heads]")
    if page_table.numel() < plan.entries(pool[3]):
        raise ValueError(f"the page table must have {plan.entries(pool[3])} entries for this plan")
    if plan.fixed_grid and torch.cuda.is_current_stream_capturing():
        plan._captured.add((pool[3], page_table.numel()))  # what updates have to fit
    q_args = ops._rows("q", q, n, Hq, D, dtype)
    if out is None:
        out = q.new_empty(n, Hq, D)
        o_args = (out.data_ptr(), Hq * D, D)
    else:
        if out.shape[0] < tokens:
            raise ValueError(f"out must hold the plan's {tokens} tokens")
        o_args = ops._rows("out", out, out.shape[0], Hq, D, dtype)
    if lse is None:
        lse = plan._f32.new_empty(n, Hq)
        l_stride = Hq
    else:
        l_stride = lse.stride(0)
        if lse.dtype != torch.float32 or lse.dim() != 2 or lse.stride(1) != 1 \
                or lse.shape[0] < tokens or lse.shape[1] != Hq:
            raise ValueError("lse must be fp32 [tokens, num_qo_heads] with a contiguous head axis")
    wide = (0, 0)
    if k_scale is not None and plan.widen:
        scratch = torch.empty((2, plan.wide_pages, Hk, 16, D), dtype=dtype, device=plan.device)
        wide = (scratch.data_ptr(), scratch.data_ptr() + scratch.numel())
    args = (*q_args, n, ops.dtype_code(q), k_pool.data_ptr(), v_pool.data_ptr(), *pool,
            ops._int32("page_table", page_table), page_table.numel(), Hq, Hk, D,
            D ** -0.5 if sm_scale is None else float(sm_scale), *plan._args, *wide, ops._at(sinks),
            _SINKS[sink_mode] if sinks is not None else 0, *o_args, lse.data_ptr(), l_stride,
            plan.status.data_ptr())
    ops._call(dev, ops.paged_attention_call, args, "d2sd_paged_attention")
    return out, lse


def rope_tables(num_positions: int, rotary_dim: int, theta: float, device, *,
                scaling: dict | None = None):
    """cos and sin tables for ``ops.append_kv``: fp32 [num_positions, rotary_dim / 2],
    angles in 64 bits, frequencies theta^(-2 i / rotary_dim). scaling: None;
    {"type": "linear", "factor": f}: frequencies divided by f;
    {"type": "yarn", "factor": f, "original": L, "beta_fast": 32, "beta_slow": 1,
    "truncate": True}: columns whose waves turn more than beta_fast times over L
    positions keep their frequency, those of fewer than beta_slow turns are divided by
    f, with a ramp between that is linear in the column, from the column of beta_fast
    turns to that of beta_slow (rounded down and up to whole ones unless ``truncate`` is
    False, as in GPT-OSS), and both tables are multiplied by 0.1 ln f + 1. Other keys are
    refused."""
    if rotary_dim <= 0 or rotary_dim % 2 or num_positions <= 0:
        raise ValueError("rope_tables: positive sizes, an even rotary_dim")
    i = torch.arange(0, rotary_dim, 2, dtype=torch.float64)
    freq = theta ** (-i / rotary_dim)
    gain = 1.0
    if scaling is not None:
        kind, known = scaling.get("type"), {"type", "factor"}
        if kind == "yarn":
            known |= {"original", "beta_fast", "beta_slow", "truncate"}
        elif kind != "linear":
            raise NotImplementedError(f"rope_tables: scaling {kind!r}")
        if not set(scaling) <= known:
            raise ValueError(f"rope_tables: {sorted(set(scaling) - known)} with scaling {kind!r}")
        f = float(scaling["factor"])
        if kind == "linear":
            freq = freq / f
        else:
            L = float(scaling["original"])

            def column(turns):  # the (real) column whose wave makes `turns` turns over L
                return rotary_dim * math.log(L / (turns * 2 * math.pi)) / (2 * math.log(theta))
            lo, hi = column(scaling.get("beta_fast", 32)), column(scaling.get("beta_slow", 1))
            if scaling.get("truncate", True):
                lo, hi = math.floor(lo), math.ceil(hi)
            lo, hi = max(lo, 0), min(hi, rotary_dim - 1)
            ramp = ((i / 2 - lo) / max(hi - lo, 1e-3)).clamp(0, 1)
            freq = freq * (1 - ramp) + freq / f * ramp
            gain = 0.1 * math.log(f) + 1.0 if f > 1 else 1.0
    angle = torch.arange(num_positions, dtype=torch.float64)[:, None] * freq[None]
    return ((angle.cos() * gain).float().to(device), (angle.sin() * gain).float().to(device))
