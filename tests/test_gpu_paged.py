"""The paged serving operators (b2_page_plan, b2_rope, b2_rope_append,
b2_attention_paged, b2_logprobs) against plain implementations in 64 bits, each
over the sizes, layouts, masks and types where it can go wrong, and a run of
them together against the same sequences in one piece."""
import math

import numpy as np
import pytest

import b2decode as b2

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

DT = {"f32": (torch.float32, b2.F32), "f16": (torch.float16, b2.F16), "bf16": (torch.bfloat16, b2.BF16)}
E32 = 2.0 ** -24  # half a step of fp32, relative


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def stream():
    return torch.cuda.current_stream().cuda_stream


def i32(a):
    return torch.as_tensor(np.asarray(a), dtype=torch.int32, device="cuda").contiguous()


# ---------------------------------------------------------------------------
# page plan
# ---------------------------------------------------------------------------

class Plan:
    """Buffers of one plan, outputs filled with a mark so that a value left alone shows."""

    def __init__(self, cached, fresh, P, max_pages, max_tokens, spare=3, seed=0, stride=None):
        g = np.random.default_rng(seed)
        cached, fresh = np.asarray(cached, np.int64), np.asarray(fresh, np.int64)
        R = len(cached)
        have = -(-np.maximum(cached, 0) // P)
        need = -(-np.maximum(cached + fresh, 0) // P) - have
        ids = g.permutation(int(np.minimum(have, max_pages).sum() + max(0, need.sum()) + spare)).astype(np.int32)
        self.table0 = np.full((R, stride or max_pages), -7, np.int32)
        at = 0
        for r in range(R):
            n = min(int(have[r]), max_pages)
            self.table0[r, :n] = ids[at:at + n]
            at += n
        self.free0 = ids[at:]
        self.cached0, self.fresh0, self.P, self.max_pages, self.cap = cached, fresh, P, max_pages, max_tokens
        self.cached, self.fresh = i32(cached), i32(fresh)
        self.free, self.n_free = i32(self.free0 if len(self.free0) else [0]), i32([len(self.free0)])
        self.table = i32(self.table0)
        mark = lambda n, t: torch.full((n,), -9, dtype=t, device="cuda")  # noqa: E731
        self.lens, self.starts, self.info = mark(R + 1, torch.int32), mark(R + 2, torch.int32), mark(5, torch.int32)
        self.slots, self.pos, self.req = mark(max_tokens + 1, torch.int64), mark(max_tokens + 1, torch.int32), mark(max_tokens + 1, torch.int32)

    def call(self):
        b2.page_plan(self.cached.data_ptr(), self.fresh.data_ptr(), len(self.cached0), self.P, self.free.data_ptr(),
                     self.n_free.data_ptr(), self.table.data_ptr(), self.table.stride(0), self.max_pages,
                     self.lens.data_ptr(), self.starts.data_ptr(), self.slots.data_ptr(), self.pos.data_ptr(),
                     self.req.data_ptr(), self.cap, self.info.data_ptr(), stream())
        return self

    def check(self, status=0):
        P, R = self.P, len(self.cached0)
        table, lens, slots, pos, req, starts = self.table0.copy(), self.cached0.copy(), [], [], [], [0] * (R + 1)
        taken = 0
        if status == 0:
            lens = self.cached0 + self.fresh0
            for r in range(R):
                have = -(-int(self.cached0[r]) // P)
                for e in range(have, -(-int(lens[r]) // P)):
                    table[r, e] = self.free0[taken]
                    taken += 1
                p = np.arange(int(self.cached0[r]), int(lens[r]))
                page = table[r, p // P].astype(np.int64)
                slots.append(np.where(page >= 0, page * P + p % P, -1))
                pos.append(p)
                req.append(np.full(len(p), r))
                starts[r + 1] = starts[r] + len(p)
        cat = lambda a, pad, n: np.concatenate([*a, np.full(n, pad)]) if a else np.full(n, pad)  # noqa: E731
        T = starts[R]
        pad = self.cap - T
        assert self.info.tolist() == [status, T, taken, 0, -9]
        assert np.array_equal(self.table.cpu().numpy(), table)
        assert self.lens.tolist() == [*lens.tolist(), -9] and self.starts.tolist() == [*starts, -9]
        assert np.array_equal(self.slots.cpu().numpy(), np.append(cat(slots, -1, pad), -9))
        assert np.array_equal(self.pos.cpu().numpy(), np.append(cat(pos, 0, pad), -9))
        assert np.array_equal(self.req.cpu().numpy(), np.append(cat(req, -1, pad), -9))


@pytest.mark.parametrize("R", [1, 2, 31, 257, 2049, 16384])
@pytest.mark.parametrize("P", [1, 7, 16, 64])
def test_page_plan(R, P):
    g = np.random.default_rng(R * 100 + P)
    top = 200 if R > 1000 else 2000
    cached = g.integers(0, top, R) * (g.random(R) < 0.8)
    fresh = np.where(g.random(R) < 0.5, 1, g.integers(0, 90, R)) * (g.random(R) < 0.8)
    cap = int(fresh.sum()) + int(g.integers(0, 70)) or 1
    p = Plan(cached, fresh, P, int((cached + fresh).max()) // P + 2, cap, seed=R, stride=int((cached + fresh).max()) // P + 5)
    p.call().check()


@pytest.mark.parametrize("case", ["no tokens", "exact fit", "page edge", "one long", "negative page"])
def test_page_plan_edges(case):
    if case == "no tokens":
        Plan([5, 0, 16], [0, 0, 0], 16, 2, 4, spare=0).call().check()
    elif case == "exact fit":  # every free page, table entry and token row used
        Plan([0, 15, 16], [32, 17, 16], 16, 2, 65, spare=0).call().check()
    elif case == "page edge":
        Plan([15, 16, 17, 31, 32], [1, 1, 1, 1, 1], 16, 4, 5).call().check()
    elif case == "one long":
        Plan([3], [1000003], 16, 62501, 1000010).call().check()
    else:  # an id below 0 in the table and in the list: no slot
        p = Plan([8, 0], [4, 20], 16, 2, 24)
        p.table0[0, 0] = -7
        p.table = i32(p.table0)
        p.free0[1] = -3
        p.free = i32(p.free0)
        p.call().check()


@pytest.mark.parametrize("status,kw", [
    (b2.PLAN_BAD_LENGTH, dict(cached=[4, -1], fresh=[1, 1])),
    (b2.PLAN_BAD_LENGTH, dict(cached=[4, 1], fresh=[1, -5])),
    (b2.PLAN_TABLE_FULL, dict(cached=[4, 60], fresh=[1, 5])),
    (b2.PLAN_TABLE_FULL, dict(cached=[4, 2**31 - 1], fresh=[1, 2**31 - 1])),
    (b2.PLAN_ROWS_FULL, dict(cached=[4, 3], fresh=[20, 5], max_tokens=24)),
    (b2.PLAN_NO_PAGES, dict(cached=[16, 3], fresh=[20, 5], n_free=1)),
    (b2.PLAN_NO_PAGES, dict(cached=[16, 3], fresh=[20, 5], n_free=-4)),
    (b2.PLAN_ROWS_FULL | b2.PLAN_NO_PAGES, dict(cached=[16, 3], fresh=[20, 5], n_free=1, max_tokens=8)),
])
def test_page_plan_that_does_not_fit(status, kw):
    """The table stays as it was and the step is empty."""
    p = Plan(np.minimum(kw["cached"], 64), [0, 0], 16, 4, kw.get("max_tokens", 40))
    p.cached0, p.fresh0 = np.asarray(kw["cached"]), np.asarray(kw["fresh"])
    p.cached, p.fresh = i32(p.cached0), i32(p.fresh0)
    p.n_free = i32([kw.get("n_free", 100)])
    p.call().check(status)


def test_page_plan_replayed():
    """A captured plan follows the lengths and the list that it finds at each replay."""
    p = Plan([0, 14], [3, 1], 16, 8, 9, spare=20)
    p.call().check()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        p.call()
    for cached, fresh in (([3, 15], [1, 1]), ([4, 16], [5, 0]), ([9, 16], [8, 9])):
        p.table0 = p.table.cpu().numpy()
        taken = int(p.info[2]) if cached != [3, 15] else sum(-(-n // 16) for n in (3, 15)) - 1
        p.free0 = p.free0[taken:]
        p.cached0, p.fresh0 = np.asarray(cached), np.asarray(fresh)
        p.cached.copy_(i32(cached))
        p.fresh.copy_(i32(fresh))
        p.free[:len(p.free0)] = i32(p.free0)
        p.n_free.copy_(i32([len(p.free0)]))
        graph.replay()
        p.check(b2.PLAN_ROWS_FULL if sum(fresh) > 9 else 0)


# ---------------------------------------------------------------------------
# rotary positions
# ---------------------------------------------------------------------------

def rotate64(x, pos, freqs, scale, rot, half):
    """x [T][heads][hd] -> the rotation in 64 bits, and the bound of its error in fp32:
    angle (64-bit product and reduction, then 24 bits of at most a quarter turn), sin and
    cos (2 steps), the factor, two products and their sum: under 8 half steps of
    (|a| + |b|) * scale, and the angle's own 2^-51 of a position in turns."""
    x = x.double()
    ang = pos.double()[:, None] * freqs[None, :]
    c, s = (f(ang)[:, None, :] * scale for f in (torch.cos, torch.sin))
    y, tol = x.clone(), torch.zeros_like(x)
    if rot:
        a, b = (x[..., :rot // 2], x[..., rot // 2:rot]) if half else (x[..., 0:rot:2], x[..., 1:rot:2])
        u, v = a * c - b * s, a * s + b * c
        t = (a.abs() + b.abs()) * scale * (8 * E32 + pos.double().abs()[:, None, None] * 2.0 ** -51 * 2 * math.pi)
        if half:
            y[..., :rot], tol[..., :rot] = torch.cat([u, v], -1), torch.cat([t, t], -1)
        else:
            y[..., :rot], tol[..., :rot] = (torch.stack(p, -1).flatten(-2) for p in ((u, v), (t, t)))
    return y, tol


def assert_within(got, want, tol, dtype):
    """|got - want| <= tol + half a step of the type (and half its smallest subnormal)."""
    fi = torch.finfo(dtype)
    err = (got.double() - want).abs()
    lim = tol + (want.abs() + tol) * half_step(dtype) + fi.tiny * fi.eps / 2
    bad = ~(err <= lim)
    assert not bool(bad.any()), (float(err.max()), int(bad.sum()), bad.nonzero()[:3].tolist())


def freqs_of(rot, theta=10000.0):
    return theta ** (-2.0 * torch.arange(rot // 2, dtype=torch.float64, device="cuda") / max(rot, 1))


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("hd,rot", [(64, 64), (128, 128), (64, 32), (80, 80), (96, 24), (256, 256), (64, 0), (64, 2),
                                    (128, 50), (6, 4), (250, 250)])
@pytest.mark.parametrize("T,top", [(1, 9), (19, 1000000), (333, 4096)])
def test_rope(dtype, half, hd, rot, T, top):
    dt, tid = DT[dtype]
    g = torch.Generator(device="cuda").manual_seed(T + hd)
    nh, nkv = 5, 2
    q = torch.randn(T, nh, hd, device="cuda", generator=g).to(dt)
    k = torch.randn(T, nkv, hd, device="cuda", generator=g).to(dt)
    pos = torch.randint(0, top, (T,), device="cuda", generator=g).to(torch.int32)
    f = freqs_of(rot)
    rows = b2.rope_rows(tid, nh, nkv, hd, rot, int(half), scale=1.25)
    qo, ko = torch.full_like(q, 7), torch.full_like(k, 7)
    b2.rope(rows, f.data_ptr() if rot else 0, pos.data_ptr(), T, q.data_ptr(), k.data_ptr(), qo.data_ptr(), ko.data_ptr(), stream())
    for x, y in ((q, qo), (k, ko)):
        assert_within(y, *rotate64(x, pos, f, 1.25, rot, half), dt)
    # in place, one of the two alone
    b2.rope(rows, f.data_ptr() if rot else 0, pos.data_ptr(), T, k=k.data_ptr(), k_out=k.data_ptr(), stream=stream())
    assert torch.equal(k, ko)


def test_rope_far_positions():
    """The largest positions, and negative ones: the angle keeps its bits."""
    pos = i32([2**31 - 1, -(2**31), -5, 2**30 + 12345, 99999999])
    f = freqs_of(64, 500000.0)
    q = torch.randn(5, 3, 64, device="cuda")
    out = torch.empty_like(q)
    b2.rope(b2.rope_rows(b2.F32, 3, 0, 64, 64), f.data_ptr(), pos.data_ptr(), 5, q.data_ptr(), q_out=out.data_ptr(), stream=stream())
    want, tol = rotate64(q, pos, f, 1.0, 64, False)
    assert_within(out, want, tol * 2, torch.float32)  # (the reference's angle, pos * f in float64, is off as far)


@pytest.mark.parametrize("dtype,cache", [("f32", "f16"), ("f32", "bf16"), ("f16", "f16"), ("bf16", "bf16")])
@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("layout", ["dense", "head-major", "fused kv"])
@pytest.mark.parametrize("hd,rot,off,T", [(64, 64, 0, 40), (128, 64, 0, 3), (64, 48, 1, 70), (8, 6, 0, 17), (256, 128, 0, 9)])
def test_rope_append(dtype, cache, half, layout, hd, rot, off, T):
    """Rows inside a wider projection (aligned and not), caches of three layouts, tokens without a slot; the
    rest of the cache stays as it was."""
    dt, tid = DT[dtype]
    ct, cid = DT[cache]
    g = torch.Generator(device="cuda").manual_seed(hd + T)
    nh, nkv, P, n_pages = 6, 3, 5, 31
    wide = torch.randn(T, off + (nh + 2 * nkv) * hd + 16, device="cuda", generator=g).to(dt)
    at = [off, off + nh * hd, off + (nh + nkv) * hd, off + (nh + 2 * nkv) * hd]
    q, k, v = (wide[:, a:b].view(T, -1, hd) for a, b in zip(at, at[1:]))
    mem = torch.full((n_pages * P * nkv * hd * 2 + 64,), 3.0, device="cuda", dtype=ct)
    if layout == "dense":
        kc, vc = (mem[i * n_pages * P * nkv * hd:][:n_pages * P * nkv * hd].view(n_pages, P, nkv, hd) for i in (0, 1))
        st = (0, 0, 0)
    elif layout == "head-major":
        kc, vc = (mem[i * n_pages * P * nkv * hd:][:n_pages * P * nkv * hd].view(n_pages, nkv, P, hd).transpose(1, 2) for i in (0, 1))
        st = kc.stride()[:3]
    else:
        kc, vc = mem[:n_pages * P * nkv * hd * 2].view(n_pages, 2, P, nkv, hd).unbind(1)
        st = kc.stride()[:3]
    kv = b2.paged_kv(kc.data_ptr(), vc.data_ptr(), cid, n_pages, P, nkv, hd, *st)
    slots = torch.randperm(n_pages * P, device="cuda", generator=g)[:T]
    slots[::7] = -1
    if T > 3:
        slots[2] = n_pages * P  # past the cache: nothing is written
    pos = torch.randint(0, 40000, (T,), device="cuda", generator=g).to(torch.int32)
    f = freqs_of(rot, 1e6)
    qo = torch.full((T, nh, hd), 9.0, device="cuda", dtype=dt)
    rows = b2.rope_rows(tid, nh, nkv, hd, rot, int(half), 0.9, *(x.stride(0) for x in (q, k, v)))
    want_k, tol = rotate64(k, pos, f, float(np.float32(0.9)), rot, half)
    b2.rope_append(rows, kv, f.data_ptr(), pos.data_ptr(), slots.data_ptr(), T, q.data_ptr(), k.data_ptr(), v.data_ptr(), qo.data_ptr(), stream())
    assert_within(qo, *rotate64(q, pos, f, float(np.float32(0.9)), rot, half), dt)
    real = (slots >= 0) & (slots < n_pages * P)
    s = slots[real]
    assert_within(kc[s // P, s % P], want_k[real], tol[real], ct)
    assert torch.equal(vc[s // P, s % P], v[real].to(ct))
    rest = torch.ones(n_pages, P, dtype=torch.bool, device="cuda")
    rest[s // P, s % P] = False
    assert bool((kc[rest] == 3).all()) and bool((vc[rest] == 3).all()) and bool((mem[-64:] == 3).all())
    # the cache alone, without q
    before = mem.clone()
    b2.rope_append(rows, kv, f.data_ptr(), pos.data_ptr(), slots.data_ptr(), T, 0, k.data_ptr(), v.data_ptr(), 0, stream())
    assert torch.equal(mem, before)


# ---------------------------------------------------------------------------
# attention over the paged cache
# ---------------------------------------------------------------------------

def attend64(q, kc, vc, table, lens, req, P, window, scale, softcap, slopes):
    """Row by row in 64 bits: out, lse, and a bound on the error of each row's out and lse.

    A score is a dot product of hd terms in fp32, of factors held to 2^-22 or better
    (2^-24 for fp16 and bf16 rows, used exactly), then scale, cap, slope and the difference
    to the maximum: off by at most D = 2^-22 sum|q k| scale (hd terms: at most hd / 8 of
    fp32's half steps more per mma step, 16 in all) + 16 half steps of the largest |score|
    and bias.  The weights are then off by e^D - 1 and the exponential's 2^-21, a sum of n
    weights by a few half steps more, so out is off by 2 (D + 2^-20) max|v| and lse by
    D + 2^-20 + 4 half steps of |lse|."""
    B, nh, hd = q.shape
    nkv = kc.shape[2]
    out = torch.zeros(B, nh, hd, dtype=torch.float64, device="cuda")
    lse = torch.full((B, nh), -math.inf, dtype=torch.float64, device="cuda")
    to, tl = torch.zeros(B, nh, dtype=torch.float64, device="cuda"), torch.zeros(B, nh, dtype=torch.float64, device="cuda")
    for b in range(B):
        n, r = int(lens[b]), b if req is None else int(req[b])
        lo = max(0, n - window) if window else 0
        if n <= 0 or r < 0:
            continue
        p = torch.arange(lo, n, device="cuda")
        page = table[r, p // P].long()
        k = kc[page, p % P].double().repeat_interleave(nh // nkv, 1)
        v = vc[page, p % P].double().repeat_interleave(nh // nkv, 1)
        s = torch.einsum("hd,lhd->hl", q[b].double(), k) * scale
        mag = torch.einsum("hd,lhd->hl", q[b].double().abs(), k.abs()) * scale
        D = mag.amax(1) * (2.0 ** -22 + 16 * E32) + 16 * E32 * s.abs().amax(1)
        if softcap:
            s = softcap * torch.tanh(s / softcap)
        if slopes is not None:
            bias = slopes.double()[:, None] * (p - (n - 1)).double()[None]
            D = D + 16 * E32 * bias.abs().amax(1)
            s = s + bias
        lse[b] = torch.logsumexp(s, 1)
        out[b] = torch.einsum("hl,lhd->hd", torch.exp(s - lse[b][:, None]), v)
        to[b] = 2 * (D + 2.0 ** -20) * v.abs().amax((0, 2))
        tl[b] = D + 2.0 ** -20 + 4 * E32 * lse[b].abs()
    return out, lse, to, tl


class Paged:
    """A cache of random pages with NaN in every place that no sequence holds."""

    def __init__(self, lens, nh, nkv, hd, P, dtype, cache, layout="dense", seed=0, extra=2, req=None, n_req=None, spread=1.0):
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.dt, self.tid = DT[dtype]
        self.ct, self.cid = DT[cache]
        self.lens, self.P, self.nh, self.nkv, self.hd, self.req = list(lens), P, nh, nkv, hd, req
        B = len(lens)
        R = n_req or B
        hold = [0] * R  # positions each table row holds
        for b in range(B):
            r = b if req is None else req[b]
            if 0 <= r < R:
                hold[r] = max(hold[r], lens[b])
        n = [-(-x // P) for x in hold]
        self.max_pages = max(n) + extra
        total = sum(n) + 3
        ids = torch.randperm(total, device="cuda", generator=g).to(torch.int32)
        self.table = torch.full((R, self.max_pages), -1, dtype=torch.int32, device="cuda")
        shape = (total, P, nkv, hd)
        if layout == "head-major":
            kc, vc = (torch.empty(total, nkv, P, hd, device="cuda", dtype=self.ct).transpose(1, 2) for _ in range(2))
        elif layout == "fused kv":
            kc, vc = torch.empty(total, 2, P, nkv, hd, device="cuda", dtype=self.ct).unbind(1)
        else:
            kc, vc = (torch.empty(shape, device="cuda", dtype=self.ct) for _ in range(2))
        kc.fill_(math.nan)
        vc.fill_(math.nan)
        at = 0
        for r in range(R):
            self.table[r, :n[r]] = ids[at:at + n[r]]
            p = torch.arange(hold[r], device="cuda")
            page = self.table[r, p // P].long()
            kc[page, p % P] = (spread * torch.randn(hold[r], nkv, hd, device="cuda", generator=g)).to(self.ct)
            vc[page, p % P] = torch.randn(hold[r], nkv, hd, device="cuda", generator=g).to(self.ct)
            at += n[r]
        self.kc, self.vc, self.total, self.R = kc, vc, total, R
        self.q = (1.5 * torch.randn(B, nh, hd, device="cuda", generator=g)).to(self.dt)

    def call(self, window=0, scale=0.0, softcap=0.0, slopes=None, len_add=0, lse=True, q=None, out=None, scratch=None, **strides):
        B = len(self.lens)
        q = self.q if q is None else q
        out = torch.full((B, self.nh, self.hd), 5.0, device="cuda", dtype=self.dt) if out is None else out
        ls = torch.full((B, self.nh), 5.0, device="cuda")
        kv = b2.paged_kv(self.kc.data_ptr(), self.vc.data_ptr(), self.cid, self.total, self.P, self.nkv, self.hd, *self.kc.stride()[:3])
        o = b2.paged_attn_opts(self.tid, self.nh, self.R, self.max_pages, len_add, window, scale, softcap,
                               0 if slopes is None else slopes.data_ptr(), **strides)
        if scratch is None:
            n = b2.attention_paged_scratch_bytes(B, self.nh, self.nkv, self.hd)
            scratch = torch.full((n,), 255, dtype=torch.uint8, device="cuda")  # (every word a NaN)
        self.lens_d = i32([n - len_add for n in self.lens])
        self.req_d = None if self.req is None else i32(self.req)
        b2.attention_paged(kv, o, q.data_ptr(), self.table.data_ptr(), self.lens_d.data_ptr(),
                           0 if self.req is None else self.req_d.data_ptr(), B, out.data_ptr(),
                           ls.data_ptr() if lse else 0, scratch.data_ptr(), stream())
        return out, ls

    def check(self, out, ls, window=0, scale=0.0, softcap=0.0, slopes=None, q=None):
        want, lse, to, tl = attend64(self.q if q is None else q, self.kc, self.vc, self.table, self.lens, self.req, self.P,
                                     window, scale or self.hd ** -0.5, softcap, slopes)
        assert_within(out, want, to[..., None].expand_as(want), self.dt)
        none = torch.isinf(lse)
        assert torch.equal(torch.isinf(ls) & (ls < 0), none)
        assert bool(((ls.double() - lse).abs() <= tl)[~none].all()), float((ls.double() - lse)[~none].abs().max())
        # the bound above holds for the worst signs; over a whole output the errors add up like a
        # random walk, so the 2-norm is held to what the roundings give on average: fp32 rows
        # 2^-19 (scores of some 10 with 2^-24 each, e^x at 2^-22), others half a step
        seen = want[~none]
        if seen.numel() > 1000:
            rel = float((out[~none].double() - seen).norm() / seen.norm())
            assert rel <= max(2.0 ** -19, half_step(self.dt)), rel


COMBOS = [("f32", "f16"), ("f32", "bf16"), ("f16", "f16"), ("bf16", "bf16")]


@pytest.mark.parametrize("dtype,cache", COMBOS)
@pytest.mark.parametrize("nh,nkv,hd", [(8, 2, 64), (14, 2, 64), (32, 8, 128), (7, 7, 128), (4, 1, 32), (10, 2, 80),
                                       (20, 1, 96), (33, 1, 128), (16, 4, 192), (6, 2, 256), (2, 1, 8)])
@pytest.mark.parametrize("lens,P", [([1], 16), ([0, 1, 2, 15, 16, 17, 63, 64, 65, 0], 16), ([130, 5, 700, 1, 64], 24), ([333], 1)])
def test_attention_paged(dtype, cache, nh, nkv, hd, lens, P):
    p = Paged(lens, nh, nkv, hd, P, dtype, cache, seed=nh + hd)
    p.check(*p.call())


@pytest.mark.parametrize("dtype,cache", COMBOS)
@pytest.mark.parametrize("nh,nkv,hd", [(16, 1, 64), (20, 1, 32), (26, 2, 40), (16, 1, 256), (20, 1, 192), (32, 2, 192), (40, 2, 256), (34, 2, 136)])
@pytest.mark.parametrize("lens,P", [([0, 1, 2, 15, 16, 17, 63, 64, 65, 0], 16), ([130, 5, 700, 1, 64], 24), ([5000, 3], 16)])
def test_attention_paged_wide_groups(dtype, cache, nh, nkv, hd, lens, P):
    """More than 8 and more than 16 query heads a KV head, below and past head dimensions of 64 and 128."""
    p = Paged(lens, nh, nkv, hd, P, dtype, cache, seed=nh + hd)
    p.check(*p.call())


@pytest.mark.parametrize("dtype,cache", COMBOS)
@pytest.mark.parametrize("nh,nkv,hd", [(16, 2, 192), (16, 2, 256), (24, 2, 256), (48, 2, 64), (24, 2, 128)])
def test_attention_paged_many_wide_heads(dtype, cache, nh, nkv, hd):
    """More heads in all than the joining launch gives a CTA each, with rows that are cut and rows that see nothing."""
    p = Paged([3000, 0, 1, 700, 40, 2000, 0] + [64, 5] * 14, nh, nkv, hd, 16, dtype, cache, seed=hd)
    p.check(*p.call())


@pytest.mark.parametrize("dtype,cache", COMBOS)
@pytest.mark.parametrize("nh,nkv,hd", [(12, 3, 128), (4, 2, 256), (14, 2, 200), (12, 1, 64), (20, 1, 128), (18, 1, 256)])
@pytest.mark.parametrize("window,softcap,alibi", [(0, 30.0, False), (1, 0.0, True), (100, 5.0, True), (333, 0.0, False)])
def test_attention_paged_masks_of_wide_heads(dtype, cache, nh, nkv, hd, window, softcap, alibi):
    """Window, cap and slopes with steps of 16 positions, tiles of 16 heads and several tiles a group."""
    p = Paged([1, 99, 100, 101, 600, 64, 0, 1500], nh, nkv, hd, 40, dtype, cache, "fused kv", seed=window + hd)
    slopes = 2.0 ** -(8.0 * torch.arange(1, nh + 1, device="cuda", dtype=torch.float32) / nh) if alibi else None
    kw = dict(window=window, softcap=softcap, slopes=slopes, scale=0.07)
    p.check(*p.call(**kw), **kw)


@pytest.mark.parametrize("dtype,cache", COMBOS)
@pytest.mark.parametrize("layout", ["head-major", "fused kv"])
@pytest.mark.parametrize("window,softcap,alibi", [(0, 30.0, False), (1, 0.0, False), (64, 0.0, True), (100, 5.0, True), (5000, 0.0, True)])
def test_attention_paged_masks(dtype, cache, layout, window, softcap, alibi):
    p = Paged([1, 99, 100, 101, 600, 64, 0, 1500], 12, 3, 64, 40, dtype, cache, layout, seed=window)
    slopes = 2.0 ** -torch.arange(1, 13, device="cuda", dtype=torch.float32) if alibi else None
    kw = dict(window=window, softcap=softcap, slopes=slopes, scale=0.11)
    p.check(*p.call(**kw), **kw)


@pytest.mark.parametrize("lens", [[32768], [20000, 3, 9000], [5000] * 40, [70] * 300, list(range(0, 400, 3)) + [9000]])
@pytest.mark.parametrize("dtype,cache", [("f32", "f16"), ("bf16", "bf16")])
def test_attention_paged_long_and_many(lens, dtype, cache):
    """One sequence cut over every CTA, ragged ones, and many short ones per CTA."""
    p = Paged(lens, 8, 2, 128, 16, dtype, cache, seed=len(lens))
    p.check(*p.call())


def test_attention_paged_thousands_of_rows():
    """More rows than threads in the scan; a wider table than it needs; no lse."""
    g = np.random.default_rng(0)
    lens = [int(n) for n in g.integers(0, 40, 3000)]
    p = Paged(lens, 4, 2, 64, 16, "bf16", "bf16")
    wide = torch.full((p.R, p.max_pages + 5), 10**9, dtype=torch.int32, device="cuda")
    wide[:, :p.max_pages] = p.table
    want = p.call()
    p.check(*want)
    p.table = wide
    out, ls = p.call(lse=False, table_stride=wide.stride(0))
    assert torch.equal(out, want[0]) and bool((ls == 5).all())


def test_attention_paged_rows_of_a_fixed_step():
    """A step of a fixed number of rows: long, short, empty, padding and bad ones side by side, more of them than
    the joining launch has CTAs."""
    g = np.random.default_rng(3)
    lens = [int(n) for n in g.integers(0, 30, 2600)]
    lens[:12] = [4000, 0, 700, 33, 2500, 0, 1, 900, 64, 0, 5, 1200]
    lens[1300:1304] = [3000, 0, 1500, 1500]
    p = Paged(lens, 12, 4, 64, 16, "bf16", "bf16", extra=0)
    good, lse = p.call()
    p.check(good, lse)
    p.req = [b if b % 3 else -1 for b in range(2600)]
    p.lens[4] = 4001 + p.max_pages * 16
    p.table[1300, 100] = p.total
    out, ls = p.call()
    live = torch.tensor([b % 3 > 0 for b in range(2600)], device="cuda")
    bad = torch.zeros_like(live)
    bad[[4, 1300]] = True
    assert bool(out[bad].isnan().all()) and bool(ls[bad].isnan().all())
    assert bool((out[~live] == 0).all()) and bool((ls[~live] == -math.inf).all())
    rest = torch.nonzero(live & ~bad)[:, 0]
    # (the shares are cut elsewhere: sums in another order)
    assert torch.equal(torch.isinf(ls[rest]), torch.isinf(lse[rest]))
    q = Paged.__new__(Paged)
    q.__dict__.update(p.__dict__)
    keep = rest.tolist()
    q.q, q.lens, q.req = p.q[rest], [lens[b] for b in keep], keep
    q.check(out[rest], ls[rest])


def test_attention_paged_a_million_rows():
    """More rows than the joining launch's CTAs list at once; three positions at most, so the whole of it is one
    tensor expression in 64 bits."""
    B, R, hd = 1_300_000, 50, 8
    g = torch.Generator(device="cuda").manual_seed(11)
    k, v = (torch.randn(R, 16, 1, hd, device="cuda", generator=g).bfloat16() for _ in range(2))
    q = torch.randn(B, 1, hd, device="cuda", generator=g).bfloat16()
    req = torch.randint(0, R, (B,), device="cuda", generator=g).to(torch.int32)
    n = (torch.randint(0, 10, (B,), device="cuda", generator=g) - 6).clamp(min=0).to(torch.int32)
    table = torch.arange(R, device="cuda", dtype=torch.int32)
    out, ls = torch.full_like(q, 5.0), torch.full((B, 1), 5.0, device="cuda")
    kv = b2.paged_kv(k.data_ptr(), v.data_ptr(), b2.BF16, R, 16, 1, hd)
    scratch = torch.full((b2.attention_paged_scratch_bytes(B, 1, 1, hd),), 255, dtype=torch.uint8, device="cuda")
    b2.attention_paged(kv, b2.paged_attn_opts(b2.BF16, 1, R, 1), q.data_ptr(), table.data_ptr(), n.data_ptr(), req.data_ptr(), B,
                       out.data_ptr(), ls.data_ptr(), scratch.data_ptr(), stream())
    kk, vv = (t[req.long(), :3, 0].double() for t in (k, v))
    s = torch.einsum("bd,bjd->bj", q[:, 0].double(), kk) * hd ** -0.5
    mag = torch.einsum("bd,bjd->bj", q[:, 0].double().abs(), kk.abs()).amax(1) * hd ** -0.5
    s = s.masked_fill(torch.arange(3, device="cuda")[None] >= n[:, None], -math.inf)
    lse = torch.logsumexp(s, 1)
    w = torch.where(n[:, None] > 0, torch.exp(s - lse[:, None]), 0.0)
    D = mag * (2.0 ** -22 + 32 * E32)  # (as in attend64)
    assert_within(out[:, 0], torch.einsum("bj,bjd->bd", w, vv), (2 * (D + 2.0 ** -20) * vv.abs().amax((1, 2)))[:, None].expand(B, hd),
                  torch.bfloat16)
    some = n > 0
    assert bool((ls[~some] == -math.inf).all())
    assert bool(((ls[:, 0].double() - lse).abs() <= D + 2.0 ** -20 + 4 * E32 * lse.abs())[some].all())


def test_attention_paged_cost_of_padding_rows():
    """16 sequences in calls of 8192 and 65536 rows, the rest padding: eight times the rows cost no more than some
    eight times as long (a joining launch whose CTAs, one to a row, each walk all rows takes 37 times)."""
    p = Paged([2001] * 16, 8, 2, 64, 16, "bf16", "bf16")

    def us(rows):
        lens, req = i32([2001] * 16 + [0] * (rows - 16)), i32(list(range(16)) + [-1] * (rows - 16))
        q = torch.zeros(rows, 8, 64, device="cuda", dtype=torch.bfloat16)
        out = torch.empty_like(q)
        kv = b2.paged_kv(p.kc.data_ptr(), p.vc.data_ptr(), p.cid, p.total, 16, 2, 64)
        o = b2.paged_attn_opts(b2.BF16, 8, 16, p.max_pages)
        scratch = torch.empty(b2.attention_paged_scratch_bytes(rows, 8, 2, 64), dtype=torch.uint8, device="cuda")
        best = math.inf
        for _ in range(8):
            a, b = (torch.cuda.Event(enable_timing=True) for _ in range(2))
            a.record()
            for _ in range(4):
                b2.attention_paged(kv, o, q.data_ptr(), p.table.data_ptr(), lens.data_ptr(), req.data_ptr(), rows, out.data_ptr(), 0,
                                   scratch.data_ptr(), stream())
            b.record()
            b.synchronize()
            best = min(best, a.elapsed_time(b) * 250)
        return best

    few, many = us(8192), us(65536)
    assert many < 16 * few, (few, many)


def test_attention_paged_window_ignores_freed_pages():
    p = Paged([1000, 130], 4, 2, 64, 16, "f16", "f16")
    want = p.call(window=100)
    p.table[0, :(900 // 16)] = -1  # given back by the server
    got = p.call(window=100)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_attention_paged_bad_rows_are_nan():
    """A page that does not exist, a length past the table: NaN in that row and in no other."""
    p = Paged([300, 300, 300, 300], 4, 2, 64, 16, "f32", "f16", extra=0)
    good, lse = p.call()
    p.table[1, 7] = p.total
    p.table[2, 18] = -1
    p.lens[3] = p.max_pages * 16 + 1
    out, ls = p.call()
    assert torch.equal(out[0], good[0]) and torch.equal(ls[0], lse[0])
    assert bool(out[1:].isnan().all()) and bool(ls[1:].isnan().all())
    p.lens[3] = 2**31 - 1
    assert bool(p.call(len_add=5)[0][3].isnan().all())
    q = Paged([50, 50, 50], 4, 2, 64, 16, "f32", "f16", req=[0, 1, -1], n_req=2)
    out, ls = q.call()
    q.check(out, ls)
    q.req = [0, 2, -(2**31)]
    out, ls = q.call()
    assert bool(out[1].isnan().all()) and bool((out[2] == 0).all()) and not bool(out[0].isnan().any())


def test_attention_paged_rows_of_a_prompt():
    """A step's token rows: lens = positions, len_add = 1, req = the token's request, -1 for padding."""
    req = [0] * 37 + [1] * 5 + [2] + [-1] * 4
    lens = list(range(1, 38)) + list(range(200, 205)) + [77] + [0] * 4
    p = Paged(lens, 8, 4, 64, 16, "bf16", "bf16", req=req, n_req=3)
    p.check(*p.call(len_add=1))


def test_attention_paged_strided_rows():
    p = Paged([40, 200, 3], 6, 3, 64, 16, "f16", "f16")
    wide = torch.randn(3, 6 * 64 + 129, device="cuda").half()
    q = wide[:, 1:1 + 6 * 64]  # rows at odd addresses
    out = torch.full((3, 6 * 64 + 7), 8.0, device="cuda", dtype=torch.float16)
    _, ls = p.call(q=q, out=out, q_stride=wide.stride(0), out_stride=out.stride(0))
    p.check(out[:, :6 * 64].view(3, 6, 64), ls, q=q.view(3, 6, 64))
    assert bool((out[:, 6 * 64:] == 8).all())


@pytest.mark.parametrize("size", [1e-20, 1e-3, 300.0, 3e4])
@pytest.mark.parametrize("cache", ["f16", "bf16"])
def test_attention_paged_range_of_q(size, cache):
    """fp32 queries far outside fp16's range keep their bits."""
    p = Paged([300, 17], 4, 2, 64, 16, "f32", cache, spread=min(1.0, 1.0 / size))
    p.q *= size
    p.check(*p.call())


@pytest.mark.parametrize("size", [1e30, 1e36, 2e37])
@pytest.mark.parametrize("cache", ["f16", "bf16"])
def test_attention_paged_largest_q(size, cache):
    """fp32 queries next to the type's largest value, with a scale that brings their scores back."""
    p = Paged([300, 17], 4, 2, 64, 16, "f32", cache, spread=0.1)
    p.q *= size
    assert bool(torch.isfinite(p.q).all())
    scale = float(np.float32(1.0 / size))
    p.check(*p.call(scale=scale), scale=scale)


def test_attention_paged_infinite_scores():
    """Keys of -inf score -inf: the others carry the row; a row of them alone is an empty one."""
    p = Paged([200, 130], 2, 1, 64, 16, "f32", "f16")
    p.q.fill_(1.0)
    pages = p.table[0].long()
    p.kc[pages[3:9], :, :, 0] = -math.inf
    pages = p.table[1].long()
    p.kc[pages[:9], :, :, 0] = -math.inf
    out, ls = p.call()
    keep = [i for i in range(200) if not 3 <= i // 16 < 9]
    k, v = (c[p.table[0, torch.tensor(keep, device="cuda") // 16].long(), torch.tensor(keep, device="cuda") % 16, 0].double() for c in (p.kc, p.vc))
    w = torch.softmax(k.sum(1) / 8, 0)
    assert float((out[0, 0].double() - w @ v).abs().max()) < 1e-4
    assert bool((out[1] == 0).all()) and bool((ls[1] == -math.inf).all())


def test_attention_paged_streams_and_graph():
    """Two calls at once with a scratch each; a captured call follows new lengths, tables and queries."""
    a = Paged([9000, 1, 300], 8, 2, 128, 16, "f32", "f16", seed=1)
    c = Paged([40, 8000], 8, 2, 128, 16, "f32", "f16", seed=2)
    wa, wc = a.call(), c.call()
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    for _ in range(5):
        with torch.cuda.stream(s1):
            ga = a.call()
        with torch.cuda.stream(s2):
            gc = c.call()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip((*ga, *gc), (*wa, *wc)))
    n = b2.attention_paged_scratch_bytes(3, 8, 2, 128)
    scratch = torch.zeros(n, dtype=torch.uint8, device="cuda")
    lens = i32([9000, 1, 300])
    out, ls = torch.empty_like(wa[0]), torch.empty_like(wa[1])
    kv = b2.paged_kv(a.kc.data_ptr(), a.vc.data_ptr(), a.cid, a.total, 16, 2, 128)
    o = b2.paged_attn_opts(b2.F32, 8, a.R, a.max_pages)

    def go():
        b2.attention_paged(kv, o, a.q.data_ptr(), a.table.data_ptr(), lens.data_ptr(), 0, 3, out.data_ptr(), ls.data_ptr(),
                           scratch.data_ptr(), stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        go()
    for new in ([9000, 1, 300], [17, 0, 299], [8999, 1, 1]):
        lens.copy_(i32(new))
        a.lens = new
        a.q.mul_(-1.0)
        graph.replay()
        a.check(out, ls)


def test_attention_paged_behind_its_plan_in_one_graph():
    """Plan, append and attention in one captured graph that also moves the lengths, the free list and the rows on:
    each replay's attention follows the lengths, requests and table entries written just before it."""
    R, P, nh, nkv, hd, cap, steps, n_pages, mp = 5, 16, 8, 2, 64, 12, 40, 64, 20
    g = torch.Generator(device="cuda").manual_seed(9)
    bank = torch.randn(steps, cap, (nh + 2 * nkv) * hd, device="cuda", generator=g).half()
    turns = [[1, 3, 0, 2, 1], [0, 1, 1, 1, 1], [2, 2, 2, 2, 2]]
    fresh_bank = i32([turns[i % 3] for i in range(steps)])
    free_all = torch.randperm(n_pages, device="cuda", generator=g).to(torch.int32)
    new = lambda *n, t=torch.int32: torch.zeros(*n, dtype=t, device="cuda")  # noqa: E731
    cached, fresh, used, at, n_free, table = new(R), new(R), new(1, t=torch.int64), new(1, t=torch.int64), new(1), new(R, mp)
    lens, starts, slots, pos, req, info = new(R), new(R + 1), new(cap, t=torch.int64), new(cap), new(cap), new(4)
    free, rows_in = new(n_pages), new(cap, (nh + 2 * nkv) * hd, t=torch.float16)
    kc, vc = (torch.full((n_pages, P, nkv, hd), math.nan, device="cuda", dtype=torch.float16) for _ in range(2))
    q, out, ls = new(cap, nh, hd, t=torch.float16), new(cap, nh, hd, t=torch.float16), new(cap, nh, t=torch.float32)
    kv = b2.paged_kv(kc.data_ptr(), vc.data_ptr(), b2.F16, n_pages, P, nkv, hd)
    rr = b2.rope_rows(b2.F16, nh, nkv, hd, 0, 0, 1.0, *[rows_in.stride(0)] * 3)
    opts = b2.paged_attn_opts(b2.F16, nh, R, mp, len_add=1)
    scratch = torch.empty(b2.attention_paged_scratch_bytes(cap, nh, nkv, hd), dtype=torch.uint8, device="cuda")
    table.fill_(-1)
    lane = torch.arange(n_pages, device="cuda")

    def step():
        fresh.copy_(fresh_bank.index_select(0, at)[0])
        rows_in.copy_(bank.index_select(0, at)[0])
        free.copy_(free_all[(lane + used).clamp(max=n_pages - 1)])
        n_free.copy_(n_pages - used)
        b2.page_plan(cached.data_ptr(), fresh.data_ptr(), R, P, free.data_ptr(), n_free.data_ptr(), table.data_ptr(), mp, mp,
                     lens.data_ptr(), starts.data_ptr(), slots.data_ptr(), pos.data_ptr(), req.data_ptr(), cap, info.data_ptr(), stream())
        e = rows_in.data_ptr()
        b2.rope_append(rr, kv, 0, pos.data_ptr(), slots.data_ptr(), cap, e, e + 2 * nh * hd, e + 2 * (nh + nkv) * hd, q.data_ptr(), stream())
        b2.attention_paged(kv, opts, q.data_ptr(), table.data_ptr(), pos.data_ptr(), req.data_ptr(), cap, out.data_ptr(), ls.data_ptr(),
                           scratch.data_ptr(), stream())
        cached.copy_(lens)
        used.add_(info[2].long())
        at.add_(1)

    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        step()  # (what the allocator needs, before the capture)
    torch.cuda.synchronize()
    for t in (cached, used, at):
        t.zero_()
    table.fill_(-1)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    held = [[] for _ in range(R)]
    for i in range(steps):
        graph.replay()
        rows, owner, length = bank[i].view(cap, nh + 2 * nkv, hd), [], []
        for r in range(R):
            for _ in range(turns[i % 3][r]):
                held[r].append(rows[len(owner), nh:])
                owner.append(r)
                length.append(len(held[r]))
        T = len(owner)
        assert info.tolist()[:2] == [0, T] and lens.tolist() == [len(h) for h in held]
        assert bool((out[T:] == 0).all()) and bool((ls[T:] == -math.inf).all())
        for r in range(R):
            if held[r]:
                p = torch.arange(len(held[r]), device="cuda")
                page, have = table[r, p // P].long(), torch.stack(held[r])
                assert torch.equal(kc[page, p % P], have[:, :nkv]) and torch.equal(vc[page, p % P], have[:, nkv:])
        p = Paged.__new__(Paged)
        p.q, p.kc, p.vc, p.table, p.lens, p.req, p.P, p.hd, p.dt = rows[:T, :nh], kc, vc, table, length, owner, P, hd, torch.float16
        p.check(out[:T], ls[:T])


def test_attention_paged_same_bits_again():
    p = Paged([5000, 77, 0, 900], 8, 2, 128, 16, "f32", "f16")
    first = p.call()
    for _ in range(3):
        assert all(torch.equal(x, y) for x, y in zip(p.call(), first))


def test_attention_paged_offsets_past_32_bits():
    """Pages whose first element lies past 2^32 elements, on a cache that is a view of 12 GB."""
    if torch.cuda.mem_get_info()[0] < 30 << 30:
        pytest.skip("needs 30 GB of free device memory")
    P, nkv, hd = 16, 8, 128
    n_pages = (2**32 + 2**31) // (P * nkv * hd)
    mem = torch.empty(n_pages, P, nkv, hd, device="cuda", dtype=torch.float16)
    p = Paged([300, 40], 8, nkv, hd, P, "f16", "f16")
    far = torch.arange(n_pages - p.total, n_pages, device="cuda")
    mem[far] = p.kc
    want = p.call()
    p.table = torch.where(p.table >= 0, p.table + (n_pages - p.total), -1).to(torch.int32)
    kc, vc, total = p.kc, p.vc, p.total
    p.kc, p.total = mem, n_pages
    p.vc = torch.empty_like(mem)
    p.vc[far] = vc
    got = p.call()
    assert all(torch.equal(x, y) for x, y in zip(got, want))
    # and written there
    k = torch.randn(1, nkv, hd, device="cuda").half()
    slot = torch.tensor([n_pages * P - 1], device="cuda")
    kv = b2.paged_kv(mem.data_ptr(), p.vc.data_ptr(), b2.F16, n_pages, P, nkv, hd)
    b2.rope_append(b2.rope_rows(b2.F16, 8, nkv, hd, 0), kv, 0, i32([3]).data_ptr(), slot.data_ptr(), 1, 0, k.data_ptr(), k.data_ptr(), 0, stream())
    assert torch.equal(mem[-1, -1], k[0]) and torch.equal(p.vc[-1, -1], k[0])


# ---------------------------------------------------------------------------
# log probabilities
# ---------------------------------------------------------------------------

def logp_call(x, dtype, n, ids, k, entropy=True):
    rows = x.shape[0]
    m = ids.shape[1]
    lp = torch.full((rows, m), 9.0, device="cuda")
    H = torch.full((rows,), 9.0, device="cuda")
    ti = torch.full((rows, k), -5, device="cuda", dtype=torch.int32)
    tl = torch.full((rows, k), 9.0, device="cuda")
    b2.logprobs(x.data_ptr(), DT[dtype][1], n, rows, x.stride(0), ids.data_ptr() if m else 0, m, lp.data_ptr() if m else 0,
                H.data_ptr() if entropy else 0, k, ti.data_ptr() if k else 0, tl.data_ptr() if k else 0, stream())
    return lp, H, ti, tl


def logp_check(x, n, ids, k, lp, H, ti, tl):
    """log S is a sum of n positive terms, each e^d at 2^-21 (the exponential and its argument),
    in at most n / 512 + 30 additions: off by at most (n / 512 + 30) half steps + 2^-21; d, the
    product and the difference add 4 half steps of |d| + |log p|."""
    d = x[:, :n].double()
    d = d - d.amax(1, keepdim=True)  # (log n is below float64's last bit of a row of the lowest fp32 value)
    ref = d - torch.logsumexp(d, 1, keepdim=True)
    sum_tol = (n / 512 + 30) * E32 + 2.0 ** -21

    def near(got, want):
        fin = torch.isfinite(want)
        assert torch.equal(got.double()[~fin], want[~fin])  # -inf where it is left out
        lim = sum_tol + 8 * E32 * want.abs()
        assert bool(((got.double() - want).abs() <= lim)[fin].all()), float((got.double() - want)[fin].abs().max())

    if ids.shape[1]:
        near(lp, torch.gather(ref, 1, ids.long()))
    if k:
        order = torch.sort(d, dim=1, descending=True, stable=True).indices[:, :k]
        assert torch.equal(ti.long(), order)
        near(tl, torch.gather(ref, 1, order))
    want = -torch.where(torch.isfinite(ref), ref.exp() * ref, 0.0).sum(1)
    # every term's weight is off as far as e^d is, and d e^d by 4 half steps of d
    lim = sum_tol * (2 + want.abs() * 2) + 8 * E32 * want.abs()
    assert bool(((H.double() - want).abs() <= lim).all()), float((H.double() - want).abs().max())


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("n", [1, 2, 31, 100, 511, 4096, 4099, 32000, 128256, 151936])
@pytest.mark.parametrize("rows,pad", [(1, 0), (3, 5), (17, 8), (80, 64)])
def test_logprobs(dtype, n, rows, pad):
    dt, _ = DT[dtype]
    g = torch.Generator(device="cuda").manual_seed(n + rows)
    x = torch.full((rows, n + pad), math.nan, device="cuda", dtype=dt)  # what lies past n is not read
    x[:, :n] = (3 * torch.randn(rows, n, device="cuda", generator=g)).to(dt)
    for k, m in ((min(20, n), 2), (min(64, n), 0), (0, 1), (1, 8)):
        ids = torch.randint(0, n, (rows, m), device="cuda", generator=g).to(torch.int32)
        logp_check(x, n, ids, k, *logp_call(x, dtype, n, ids, k))


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("n", [1000, 40000])
def test_logprobs_many_given_tokens(dtype, n):
    """More given tokens than two for each thread, the last ones out of range."""
    dt, _ = DT[dtype]
    g = torch.Generator(device="cuda").manual_seed(n)
    x = torch.randn(3, n, device="cuda", generator=g).to(dt)
    for m in (257, 513, 1400):
        ids = torch.randint(0, n, (3, m), device="cuda", generator=g).to(torch.int32)
        lp, H, ti, tl = logp_call(x, dtype, n, ids, 5)
        logp_check(x, n, ids, 5, lp, H, ti, tl)
        ids[:, -1], ids[0, m // 2] = n, -1
        out = logp_call(x, dtype, n, ids, 5)[0]
        bad = (ids < 0) | (ids >= n)
        assert bool(out[bad].isnan().all()) and torch.equal(out[~bad], lp[~bad])


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("n", [5, 4097, 50257, 128256])
@pytest.mark.parametrize("rows", [1, 3])
def test_logprobs_rows_off_16_bytes(dtype, n, rows):
    """Logits that start at any element: one row and several, in a leading dimension of any width."""
    dt, _ = DT[dtype]
    g = torch.Generator(device="cuda").manual_seed(n + rows)
    for off, pad in ((1, 0), (2, 8), (3, 3)):
        mem = torch.full((off + rows * (n + pad) + 9,), math.nan, device="cuda", dtype=dt)
        x = mem[off:off + rows * (n + pad)].view(rows, n + pad)
        x[:, :n] = (3 * torch.randn(rows, n, device="cuda", generator=g)).to(dt)
        ids = torch.randint(0, n, (rows, 2), device="cuda", generator=g).to(torch.int32)
        logp_check(x, n, ids, min(5, n), *logp_call(x, dtype, n, ids, min(5, n)))


def test_logprobs_many_rows():
    x = torch.randn(5000, 1000, device="cuda").bfloat16()
    ids = torch.randint(0, 1000, (5000, 1), device="cuda").to(torch.int32)
    logp_check(x, 1000, ids, 5, *logp_call(x, "bf16", 1000, ids, 5))


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("kind", ["zeros", "signed zeros", "two levels", "lowest value", "lowest and -inf", "few allowed", "one allowed", "ascending",
                                  "descending", "one thread", "runs", "large", "tail"])
@pytest.mark.parametrize("n", [700, 20011, 131072, 300001])
@pytest.mark.parametrize("rows", [1, 100])
def test_logprobs_ties_and_masks(dtype, kind, n, rows):
    """Alternatives where very many logits are equal, masked, in order, or in one thread's hands."""
    dt, _ = DT[dtype]
    g = torch.Generator(device="cuda").manual_seed(n)
    x = torch.zeros(rows, n, device="cuda")
    i = torch.arange(n, device="cuda")
    some = torch.randperm(n, device="cuda", generator=g)
    if kind == "signed zeros":
        x[:, ::2] = -0.0
    elif kind == "two levels":
        x[:, some[:n // 3]] = 1.0
    elif kind == "lowest value":  # a mask of the type's lowest value, seven allowed
        x.fill_(torch.finfo(dt).min)
        x[1 if rows > 1 else 0:, some[:7]] = torch.randn(7, device="cuda", generator=g)  # (row 0 of many: nothing allowed)
    elif kind == "lowest and -inf":
        x.fill_(-math.inf)
        x[:, some[:n // 2]] = torch.finfo(dt).min
    elif kind == "few allowed":
        x.fill_(-math.inf)
        x[:, some[:7]] = torch.randn(rows, 7, device="cuda", generator=g)
    elif kind == "one allowed":
        x.fill_(-math.inf)
        x[:, some[0]] = -3.0
    elif kind in ("ascending", "descending"):
        x[:] = (i if kind == "ascending" else n - i).float() / n * 20
    elif kind == "one thread":  # large logits 4096 apart and in long runs
        x[:, (i // 8) % 512 == 5] = 4.0 + torch.rand(int(((i // 8) % 512 == 5).sum()), device="cuda", generator=g)
    elif kind == "runs":  # a few batches of a thread hold many logits over the bound each
        x[:, (i // 8) % 256 < 40] = 4.0 + torch.rand(int(((i // 8) % 256 < 40).sum()), device="cuda", generator=g)
    elif kind == "large":
        x[:] = 30000.0 * torch.randn(rows, n, device="cuda", generator=g).clamp(-2, 2)
    elif kind == "tail":
        x[:, -3:] = torch.tensor([5.0, 9.0, 7.0], device="cuda")
    x = x.to(dt)
    ids = torch.stack([some[0].expand(rows), some[-1].expand(rows)], 1).to(torch.int32)
    for k in (1, 20, 64):
        logp_check(x, n, ids, k, *logp_call(x, dtype, n, ids, k))


def test_logprobs_bad_rows():
    """NaN, +inf, nothing left, ids out of range: NaN there, and the other rows untouched."""
    x = torch.randn(6, 5000, device="cuda")
    ref = x.clone()
    x[1, 77] = math.nan
    x[2, 4000] = math.inf
    x[3] = -math.inf
    x[4] = math.nan
    ids = i32([[3, 5000]] * 5 + [[-1, 2**31 - 1]])
    lp, H, ti, tl = logp_call(x, "f32", 5000, ids, 8)
    for r in (1, 2, 3, 4):
        assert bool(lp[r].isnan().all()) and bool(H[r].isnan()) and bool(tl[r].isnan().all())
    assert not bool((ti[1] == 77).any()) and int(ti[2, 0]) == 4000
    assert ti[3].tolist() == list(range(8)) and ti[4].tolist() == [-1] * 8
    assert not bool(lp[0, 0].isnan()) and bool(lp[0, 1].isnan()) and bool(lp[5].isnan().all())
    logp_check(ref[[0, 5]], 5000, i32([[3], [0]])[:, :0], 8, lp[[0, 5], :0], H[[0, 5]], ti[[0, 5]], tl[[0, 5]])


def test_logprobs_outputs_left_out_and_graph():
    x = torch.randn(2, 9000, device="cuda")
    ids = i32([[4], [8999]])
    lp, H, _, _ = logp_call(x, "f32", 9000, ids, 0, entropy=False)
    assert bool((H == 9).all()) and bool((lp < 0).all())
    b2.logprobs(x.data_ptr(), b2.F32, 9000, 2, 9000, 0, 0, 0, 0, 0, 0, 0)  # nothing asked for
    out = logp_call(x, "f32", 9000, ids, 5)
    lp, H, ti, tl = (torch.empty_like(t) for t in out)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        b2.logprobs(x.data_ptr(), b2.F32, 9000, 2, 9000, ids.data_ptr(), 1, lp.data_ptr(), H.data_ptr(), 5, ti.data_ptr(), tl.data_ptr(), stream())
    for _ in range(3):
        x.normal_()
        graph.replay()
        logp_check(x, 9000, ids, 5, lp, H, ti, tl)


@pytest.mark.parametrize("graph", [False, True])
def test_batch_scores(built_lib, write_model, graph):
    """The batched decode's own logits, scored in place: equal to the scores of the copied logits."""
    from b2decode import gguf_writer as gw
    shape = gw.ModelShape("qwen2", 256, 2, 4, 2, 512, 512, 256, 1e-6, 1e6, True, True, "q8_0", 1, 2)
    m = b2.Model(write_model("qwen2-hd64-q8", shape), num_ctx=64)
    bt = b2.Batch(m, 3)
    bt.use_graph(graph)
    nxt = [bt.prefill(i, [1, 5 + i, 9]) for i in range(3)]
    first = bt.logprobs([[nxt[2], 3]], 5)  # after a prefill: its last token
    x = torch.from_numpy(bt.logits()[:1]).cuda()
    check = lambda x, ids, r: logp_check(x, 512, i32(ids), r[2].shape[1], *(torch.from_numpy(t).cuda() for t in r))  # noqa: E731
    check(x, [[nxt[2], 3]], first)
    assert first[2][0, 0] == nxt[2]
    for _ in range(4):
        nxt = bt.step(nxt)
        got = bt.logprobs(np.asarray(nxt)[:, None], 4)
        check(torch.from_numpy(bt.logits()).cuda(), np.asarray(nxt)[:, None], got)
        assert np.array_equal(got[2][:, 0], nxt) and np.array_equal(got[0][:, 0], got[3][:, 0])
    assert bt.logprobs(np.zeros((3, 0)), 0)[1].shape == (3,)
    for rows, top in ((4, 1), (3, 65)):
        with pytest.raises(b2.B2Error, match="b2_batch_logprobs"):
            bt.logprobs(np.zeros((rows, 1)), top)
    bt.close()
    m.close()


def test_batch_scores_of_rows_that_no_forward_left(built_lib, write_model):
    """More rows than the last forward's logits: refused, not scores of an older step."""
    from b2decode import gguf_writer as gw
    shape = gw.ModelShape("qwen2", 256, 2, 4, 2, 512, 512, 256, 1e-6, 1e6, True, True, "q8_0", 1, 2)
    m = b2.Model(write_model("qwen2-hd64-q8", shape), num_ctx=16)
    bt = b2.Batch(m, 2)

    def refused(rows, left):
        with pytest.raises(b2.B2Error, match="b2_batch_logprobs: the last forward left %d rows" % left) as e:
            bt.logprobs(np.zeros((rows, 1)), 1)
        assert e.value.code == -8

    refused(1, 0)
    nxt = [bt.prefill(i, [1, 5 + i]) for i in range(2)]
    refused(2, 1)
    assert bt.logprobs([[nxt[1]]], 1)[2][0, 0] == nxt[1]
    nxt = bt.step(nxt)
    assert np.array_equal(bt.logprobs(np.zeros((2, 1)), 1)[2][:, 0], nxt)
    with pytest.raises(b2.B2Error):  # a prompt that is refused leaves the step's logits
        bt.prefill(0, list(range(1, 17)))
    assert np.array_equal(bt.logprobs(np.zeros((2, 1)), 1)[2][:, 0], nxt)
    bt.prefill(0, [1, 5, 6])
    refused(2, 1)
    bt.close()
    m.close()


@pytest.mark.skipif(torch.cuda.device_count() < 2, reason="needs a second device to be current")
def test_batch_scores_with_another_device_current(built_lib, write_model):
    """Refused as a step and a prefill are, before anything is launched."""
    from b2decode import gguf_writer as gw
    shape = gw.ModelShape("qwen2", 256, 2, 4, 2, 512, 512, 256, 1e-6, 1e6, True, True, "q8_0", 1, 2)
    m = b2.Model(write_model("qwen2-hd64-q8", shape), num_ctx=64)
    bt = b2.Batch(m, 1)
    first = bt.prefill(0, [1, 5, 9])
    with torch.cuda.device(1):
        with pytest.raises(b2.B2Error, match="must be the current device") as e:
            bt.logprobs([[first]], 1)
        assert e.value.code == -8
    assert bt.logprobs([[first]], 1)[2][0, 0] == first
    bt.close()
    m.close()


# ---------------------------------------------------------------------------
# refusals that need a device, and a run of all of them
# ---------------------------------------------------------------------------

def test_host_memory_is_refused():
    x = torch.randn(2, 100)
    d = torch.randn(2, 100, device="cuda")
    with pytest.raises(b2.B2Error, match="not device memory"):
        b2.logprobs(x.data_ptr(), b2.F32, 100, 2, 100, 0, 0, 0, d.data_ptr(), 0, 0, 0)
    with pytest.raises(b2.B2Error, match="not device memory"):
        b2.rope(b2.rope_rows(b2.F32, 1, 0, 100, 0), 0, i32([0, 0]).data_ptr(), 2, d.data_ptr(), q_out=x.data_ptr())


@pytest.mark.parametrize("P", [16, 24])
def test_a_served_run(P):
    """Five requests from prompts of 0 to 70 tokens through ten steps of a one-layer model with pages
    handed out as they grow, one request joining and one leaving on the way: every step's outputs
    and scores equal those of the same sequences kept in one piece, in 64 bits."""
    g = torch.Generator(device="cuda").manual_seed(P)
    nh, nkv, hd, V, R, cap = 8, 2, 64, 5000, 5, 160
    H = nh * hd
    emb = torch.randn(V, H, device="cuda", generator=g)
    wqkv = torch.randn(H, (nh + 2 * nkv) * hd, device="cuda", generator=g) / H ** 0.5
    head = torch.randn(H, V, device="cuda", generator=g) / H ** 0.5
    f, scale = b2.rope_freqs(hd, 10000.0, b2.ROPE_SCALE_YARN, 4.0, 64.0)
    fd = torch.from_numpy(f).cuda()
    n_pages = 60
    cache = torch.full((n_pages, 2, P, nkv, hd), math.nan, device="cuda", dtype=torch.float16)
    kc, vc = cache.unbind(1)
    kv = b2.paged_kv(kc.data_ptr(), vc.data_ptr(), b2.F16, n_pages, P, nkv, hd, *kc.stride()[:3])
    max_pages = 12
    table = torch.full((R, max_pages), -1, dtype=torch.int32, device="cuda")
    free = list(np.random.default_rng(P).permutation(n_pages))
    rows = b2.rope_rows(b2.F32, nh, nkv, hd, hd, b2.ROPE_HALF, scale, *[(nh + 2 * nkv) * hd] * 3)
    opts = b2.paged_attn_opts(b2.F32, nh, R, max_pages, len_add=1, softcap=20.0, window=90)
    scratch = torch.empty(b2.attention_paged_scratch_bytes(cap, nh, nkv, hd), dtype=torch.uint8, device="cuda")
    new = lambda n, t=torch.int32: torch.empty(n, dtype=t, device="cuda")  # noqa: E731
    lens, starts, slots, pos, req, info = new(R), new(R + 1), new(cap, torch.int64), new(cap), new(cap), new(4)
    attn, lp, ent, ti, tl = (torch.empty(cap, H, device="cuda"), torch.empty(cap, 1, device="cuda"),
                             torch.empty(cap, device="cuda"), new((cap, 4)), torch.empty(cap, 4, device="cuda"))
    rng = np.random.default_rng(P + 1)
    text = [[int(t) for t in rng.integers(0, V, n)] for n in (70, 1, 33, 0, 20)]
    cached, joined = [0] * R, [True, True, True, False, True]
    for step in range(10):
        if step == 4:  # request 3 joins with a prompt, request 0 leaves and gives its pages back
            text[3], joined[3] = [int(t) for t in rng.integers(0, V, 45)], True
            free = [int(p) for p in table[0].tolist() if p >= 0] + free
            table[0] = -1
            text[0], cached[0], joined[0] = [], 0, False
        fresh = [len(t) - c if j else 0 for t, c, j in zip(text, cached, joined)]
        toks = [t for r in range(R) for t in text[r][cached[r]:cached[r] + fresh[r]]]
        T = len(toks)
        free_d, n_free, cd, fr = i32(free), i32([len(free)]), i32(cached), i32(fresh)
        b2.page_plan(cd.data_ptr(), fr.data_ptr(), R, P, free_d.data_ptr(), n_free.data_ptr(), table.data_ptr(), max_pages, max_pages,
                     lens.data_ptr(), starts.data_ptr(), slots.data_ptr(), pos.data_ptr(), req.data_ptr(), cap, info.data_ptr(), stream())
        x = torch.zeros(cap, H, device="cuda")
        x[:T] = emb[torch.tensor(toks, device="cuda")]
        qkv = x @ wqkv
        q, k, v = qkv[:, :H], qkv[:, H:H + nkv * hd], qkv[:, H + nkv * hd:]
        raw = qkv.clone()
        b2.rope_append(rows, kv, fd.data_ptr(), pos.data_ptr(), slots.data_ptr(), cap, q.data_ptr(), k.data_ptr(), v.data_ptr(),
                       attn.data_ptr(), stream())
        rot = attn.clone()
        b2.attention_paged(kv, opts, rot.data_ptr(), table.data_ptr(), pos.data_ptr(), req.data_ptr(), cap, attn.data_ptr(), 0,
                           scratch.data_ptr(), stream())
        logits = attn @ head
        nxt = torch.argmax(logits, 1).to(torch.int32)
        b2.logprobs(logits.data_ptr(), b2.F32, V, cap, V, nxt.data_ptr(), 1, lp.data_ptr(), ent.data_ptr(), 4, ti.data_ptr(),
                    tl.data_ptr(), stream())
        status = info.tolist()
        assert status[:2] == [0, T]
        free = free[status[2]:]
        # the same rows with each sequence in one piece
        assert bool((attn[T:] == 0).all())
        for r in range(R):
            if not fresh[r]:
                continue
            seq = emb[torch.tensor(text[r], device="cuda")] @ wqkv
            p = torch.arange(len(text[r]), device="cuda")
            qq, kk, vv = (seq[:, a:b].reshape(len(p), -1, hd) for a, b in ((0, H), (H, H + nkv * hd), (H + nkv * hd, seq.shape[1])))
            qq, kk = (rotate64(t, p, fd, float(np.float32(scale)), hd, True)[0] for t in (qq, kk))
            kk, vv = (t.half().double().repeat_interleave(nh // nkv, 1) for t in (kk, vv))
            s = 20 * torch.tanh(torch.einsum("ihd,jhd->hij", qq, kk) / 8 / 20)
            dist = p[:, None] - p[None, :]
            s = s.masked_fill((dist < 0) | (dist >= 90), -math.inf)
            want = torch.einsum("hij,jhd->ihd", torch.softmax(s, 2), vv).reshape(len(p), H)[cached[r]:]
            a = int(starts[r])
            got = attn[a:a + fresh[r]].double()
            # the two sides' fp32 projections may differ in the last bits, and with them an fp16 key's rounding
            assert float((got - want).norm() / want.norm()) < 2.0 ** -11
            full = torch.log_softmax(logits[a:a + fresh[r]].double(), 1)
            best = full.max(1)
            assert torch.equal(ti[a:a + fresh[r], 0].long(), best.indices) and torch.equal(lp[a:a + fresh[r], 0], tl[a:a + fresh[r], 0])
            assert float((lp[a:a + fresh[r], 0].double() - best.values).abs().max()) < 1e-5
            assert float((ent[a:a + fresh[r]].double() + (full.exp() * full).sum(1)).abs().max()) < 1e-4
            cached[r] += fresh[r]
            text[r].append(int(nxt[a + fresh[r] - 1]))
        del raw
