"""Attention of rows that share a prefix (b2_attention_shared) against the
same rows one by one in 64 bits: groups of every size, lengths on and around
the tiles' and pages' edges, masks that leave a row nothing, values that one row
of a group sees and another does not."""
import math

import numpy as np
import pytest

import b2decode as b2
from test_gpu_paged import COMBOS, DT, Paged, assert_within, attend64, half_step, i32, stream

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


class Shared(Paged):
    """Groups [(rows' lengths, shared positions)]; a length below 0 is a row without a sequence.  The rows of a
    group have table rows of their own (the pages of the shared positions the same) or, with `one`, are tokens of
    one sequence.  NaN in every place that no row sees.  `wide`: a table with room for so many positions that the
    rows are taken together (small calls run row by row)."""

    def __init__(self, groups, nh, nkv, hd, P, dtype, cache, layout="dense", seed=0, one=False, alone=(), wide=True):
        lens = [max(n, 0) for ls, _ in groups for n in ls] + list(alone)
        at, req = 0, []
        for i, (ls, _) in enumerate(groups):
            req += [i if one and n >= 0 else at + j if n >= 0 else -1 for j, n in enumerate(ls)]
            at += len(ls)
        req += [len(groups) + i if one else at + i for i in range(len(alone))]
        super().__init__(lens, nh, nkv, hd, P, dtype, cache, layout, seed, req=req, n_req=max(max(req) + 1, 1))
        self.sizes = [len(ls) for ls, _ in groups]
        self.starts, self.prefix = np.cumsum([0] + self.sizes), [p for _, p in groups]
        if not one:  # the later rows' pages of the shared positions are the first row's
            at = 0
            for ls, p in groups:
                rows = [at + j for j, n in enumerate(ls) if n >= 0]
                if rows:
                    first = max(rows, key=lambda r: lens[r])
                    for r in rows:
                        n = min(-(-min(lens[r], p) // P), -(-lens[first] // P))
                        self.table[r, :n] = self.table[first, :n]
                at += len(ls)
        if wide:
            per = len(lens) * P * nkv * max(nh // nkv, 8) * hd
            self.max_pages = max(self.max_pages, 2 ** 28 // per + 1)
            table = torch.full((self.R, self.max_pages), -1, dtype=torch.int32, device="cuda")
            table[:, :self.table.shape[1]] = self.table
            self.table = table

    def call(self, window=0, scale=0.0, softcap=0.0, slopes=None, len_add=0, lse=True, q=None, out=None, scratch=None,
             starts=None, prefix=None, n_groups=None, **strides):
        B = len(self.lens)
        q = self.q if q is None else q
        out = torch.full((B, self.nh, self.hd), 5.0, device="cuda", dtype=self.dt) if out is None else out
        ls = torch.full((B, self.nh), 5.0, device="cuda")
        kv = b2.paged_kv(self.kc.data_ptr(), self.vc.data_ptr(), self.cid, self.total, self.P, self.nkv, self.hd, *self.kc.stride()[:3])
        o = b2.paged_attn_opts(self.tid, self.nh, self.R, self.max_pages, len_add, window, scale, softcap,
                               0 if slopes is None else slopes.data_ptr(), **strides)
        if scratch is None:
            n = b2.attention_shared_scratch_bytes(B, self.nh, self.nkv, self.hd)
            scratch = torch.full((n,), 255, dtype=torch.uint8, device="cuda")
        self.lens_d = i32([n - len_add for n in self.lens])
        self.req_d = i32(self.req)
        self.starts_d, self.prefix_d = i32(self.starts if starts is None else starts), i32(self.prefix if prefix is None else prefix)
        b2.attention_shared(kv, o, q.data_ptr(), self.table.data_ptr(), self.lens_d.data_ptr(), self.req_d.data_ptr(), B,
                            self.starts_d.data_ptr(), self.prefix_d.data_ptr(), n_groups or len(self.prefix_d), out.data_ptr(),
                            ls.data_ptr() if lse else 0, scratch.data_ptr(), stream())
        self.scratch = scratch
        return out, ls


    def check(self, out, ls, window=0, scale=0.0, softcap=0.0, slopes=None, q=None):
        """As Paged.check, with the rounding of 16-bit rows' probabilities to one 16-bit term: each weight off by at
        most half a step h, so out = sum w v / sum w by at most h max|v|.  (Averaged over a whole output that error
        is as large as the rounding of the result, sqrt(2) together, well inside the half step that the 2-norm gets.)"""
        want, lse, to, tl = attend64(self.q if q is None else q, self.kc, self.vc, self.table, self.lens, self.req, self.P,
                                     window, scale or self.hd ** -0.5, softcap, slopes)
        h = half_step(self.dt) if self.dt != torch.float32 else 0.0
        to = to + h * float(torch.nan_to_num(self.vc.float(), 0.0, 0.0, 0.0).abs().max())
        assert_within(out, want, to[..., None].expand_as(want), self.dt)
        none = torch.isinf(lse)
        assert torch.equal(torch.isinf(ls) & (ls < 0), none)
        assert bool(((ls.double() - lse).abs() <= tl)[~none].all()), float((ls.double() - lse)[~none].abs().max())
        seen = want[~none]
        if seen.numel() > 1000:
            rel = float((out[~none].double() - seen).norm() / seen.norm())
            assert rel <= max(2.0 ** -19, half_step(self.dt)), rel


@pytest.mark.parametrize("dtype,cache", COMBOS)
@pytest.mark.parametrize("nh,nkv,hd", [(8, 2, 64), (14, 2, 64), (32, 8, 128), (7, 7, 128), (4, 1, 32), (10, 2, 80), (20, 1, 96),
                                       (33, 1, 128), (2, 1, 8), (3, 1, 120), (6, 2, 256), (130, 1, 64), (256, 1, 72)])
@pytest.mark.parametrize("groups,P", [
    ([([1], 1)], 16),
    ([([40, 41, 50, 40], 40)], 16),
    ([([130, 131, 300, 129], 128), ([5], 0), ([0, 0], 0), ([64, 20, -1, 65], 64)], 24),
    ([([700] * 9, 700), ([333, 257, 256, 255, 1, 0], 256)], 1)])
def test_attention_shared(dtype, cache, nh, nkv, hd, groups, P):
    for wide in (True, False):
        p = Shared(groups, nh, nkv, hd, P, dtype, cache, seed=nh + hd, wide=wide)
        p.check(*p.call())


@pytest.mark.parametrize("dtype,cache", COMBOS)
@pytest.mark.parametrize("nh,nkv,hd", [(8, 1, 128), (14, 2, 64)])
@pytest.mark.parametrize("n", [1, 2, 15, 16, 17, 31, 32, 33, 127, 128, 129, 255, 256, 257, 385])
def test_attention_shared_lengths(dtype, cache, nh, nkv, hd, n):
    """Shared and own parts of every length around the edges of products, loads and tiles."""
    g = [([n + s for s in (0, 1, 17, 128, 129)], n), ([n, n], n), ([n + 3], 0)]
    p = Shared(g, nh, nkv, hd, 16, dtype, cache, seed=n)
    p.check(*p.call())


@pytest.mark.parametrize("dtype,cache", COMBOS)
@pytest.mark.parametrize("tokens,total", [(1, 1), (5, 5), (130, 130), (300, 511), (33, 2000), (2, 129)])
@pytest.mark.parametrize("nh,nkv,hd", [(8, 1, 128), (14, 2, 64), (4, 4, 96)])
def test_attention_shared_prompt(dtype, cache, tokens, total, nh, nkv, hd):
    """The last tokens of a sequence as the rows of a group: each sees the positions up to its own."""
    lens = [total - tokens + 1 + i for i in range(tokens)]
    p = Shared([(lens, total), ([7, 8, 9], 9), ([300], 300)], nh, nkv, hd, 16, dtype, cache, seed=tokens, one=True)
    p.check(*p.call())


@pytest.mark.parametrize("dtype,cache", COMBOS)
@pytest.mark.parametrize("layout", ["head-major", "fused kv"])
@pytest.mark.parametrize("window,softcap,alibi", [(0, 30.0, False), (1, 0.0, False), (64, 0.0, True), (100, 5.0, True),
                                                  (300, 0.0, False), (5000, 0.0, True)])
@pytest.mark.parametrize("one", [False, True])
def test_attention_shared_masks(dtype, cache, layout, window, softcap, alibi, one):
    g = [([560, 600, 571, 562, 900], 560), ([1, 99, 100, 101, 64, 0, 500], 100), ([301 + i for i in range(40)], 340)]
    p = Shared(g, 12, 3, 64, 40, dtype, cache, layout, seed=window, one=one)
    slopes = 2.0 ** -torch.arange(1, 13, device="cuda", dtype=torch.float32) if alibi else None
    kw = dict(window=window, softcap=softcap, slopes=slopes, scale=0.11)
    p.check(*p.call(**kw), **kw)


@pytest.mark.parametrize("dtype,cache", [("f32", "f16"), ("bf16", "bf16")])
@pytest.mark.parametrize("groups", [
    [([32768 + i for i in range(4)], 32768)], [([4000 + 3 * i for i in range(100)], 4000)],
    [([50 * i + j for j in range(8)], 50 * i) for i in range(1, 40)], [([60 + i % 7], 0) for i in range(300)],
    [([9000] * 3, 9000), ([10] * 500, 8)]])
def test_attention_shared_long_and_many(dtype, cache, groups):
    p = Shared(groups, 8, 2, 128, 16, dtype, cache, seed=len(groups))
    p.check(*p.call())


def test_attention_shared_thousands_of_rows():
    """More rows than the laying of the line takes at once, groups across its edges, rows in no group."""
    g = np.random.default_rng(0)
    groups = []
    while sum(len(ls) for ls, _ in groups) < 3000:
        p = int(g.integers(0, 40))
        groups.append(([p + int(x) for x in g.integers(0, 9, int(g.integers(1, 400)))], p))
    p = Shared(groups, 4, 2, 64, 16, "bf16", "bf16", alone=(33, 0, 5))
    p.check(*p.call())
    p.starts = np.array(p.starts) + 2  # two rows before the first group; the last group's end is beyond the others' rows
    p.starts[-1] = len(p.lens)
    p.prefix = [0] * len(p.prefix)
    p.check(*p.call())


def test_attention_shared_thousands_of_groups():
    """More groups than the laying of the line keeps at once, of up to five rows or none."""
    groups = [([40 + i % 5, 45, 33, 50, 41][:i % 6], 30 + i % 13) for i in range(2400)]
    p = Shared(groups, 2, 1, 64, 16, "bf16", "bf16")
    assert len(p.lens) >= 2 * len(groups)
    p.check(*p.call())


def test_attention_shared_equals_paged():
    """The same numbers as b2_attention_paged to the rounding of the sums, whatever the groups say is shared."""
    p = Shared([([513 + 5 * i for i in range(20)], 512), ([40], 40)], 16, 4, 128, 16, "f32", "f16")
    a, la = Paged.call(p)
    for prefix in ([512, 40], [500, 3], [0, 0], [1, 1], [-5, 10 ** 9]):
        o, ls = p.call(prefix=prefix)
        if prefix[0] >= 0:
            assert float((o - a).norm() / a.norm()) < 2.0 ** -19 and float((ls - la).abs().max()) < 2.0 ** -17
    p.call(prefix=[512, 40])
    p.check(*p.call(prefix=[512, 40]))


@pytest.mark.parametrize("dtype,cache", COMBOS)
@pytest.mark.parametrize("window,rows", [(64, 700), (300, 150)])
@pytest.mark.parametrize("one", [False, True])
def test_attention_shared_windows(dtype, cache, window, rows, one):
    """Windows in rows enough that they are taken together; pages below every window of a group are not looked at."""
    lens = [900 + i % 97 for i in range(rows - 60)] if not one else [310 + i for i in range(rows - 60)]
    groups = [(lens, 890 if not one else max(lens)), ([200 + i for i in range(50)], 250), ([5] * 9 + [0], 5)]
    p = Shared(groups, 96, 12, 64, 16, dtype, cache, one=one)
    for r in range(p.R):  # (a table row of the first group)
        if (r == 0) if one else r < len(lens):
            p.table[r, :(min(lens) - window) // 16] = 10 ** 6
    p.check(*p.call(window=window), window=window)


def test_attention_shared_values_that_others_do_not_see():
    """Infinite and NaN values among what one row sees stay out of the rows of its group that do not see them."""
    lens = [100, 128, 200, 90, 330]
    for one in (False, True):
        p = Shared([(lens, 330)], 8, 2, 64, 16, "bf16", "bf16", one=one)
        page = lambda pos: (int(p.table[0 if one else 4, pos // 16]), pos % 16)  # noqa: E731
        p.vc[page(150)] = math.nan
        p.vc[page(110)][0, 3] = math.inf
        p.kc[page(120)][1] = math.nan
        o, ls = p.call()
        want, lse, to, tl = attend64(p.q, p.kc, p.vc, p.table, p.lens, p.req, 16, 0, 64 ** -0.5, 0.0, None)
        to = to + half_step(p.dt) * float(torch.nan_to_num(p.vc.float(), 0.0, 0.0, 0.0).abs().max())
        for b in (0, 3):  # see none of it
            assert_within(o[b], want[b], to[b][:, None].expand_as(want[b]), p.dt)
        assert bool(torch.isfinite(ls[[0, 3]]).all())
        assert torch.equal(torch.isnan(o), torch.isnan(want)) and torch.equal(torch.isinf(o), torch.isinf(want))
        ok = torch.isfinite(want)
        assert_within(o[ok], want[ok], to[..., None].expand_as(want)[ok], p.dt)


def test_attention_shared_window_ignores_freed_pages():
    p = Shared([([800, 810, 805], 800)], 8, 2, 64, 16, "bf16", "bf16")
    want = p.call(window=100)[0].clone()
    p.table[:, :40] = 10 ** 6
    o, ls = p.call(window=100)
    assert torch.equal(o, want)


def test_attention_shared_bad_rows_are_nan():
    """A length past the table, a request past it, a page past the cache: NaN where it is seen, all else untouched."""
    p = Shared([([300, 200, 40, 301], 300), ([90, 95], 90), ([20, 21], 20)], 8, 2, 64, 16, "f32", "f16", one=True)
    want, lw = (t.clone() for t in p.call())
    keep = p.table.clone()
    p.table[0, 15] = -1  # positions 240 .. 255: rows 0 and 3
    p.table[1, 0] = p.total
    o, ls = p.call()
    bad = torch.tensor([True, False, False, True, True, True, False, False], device="cuda")
    assert bool(torch.isnan(o[bad]).all()) and bool(torch.isnan(ls[bad]).all())
    assert torch.equal(o[~bad], want[~bad]) and torch.equal(ls[~bad], lw[~bad])
    p.table = keep
    p.req, p.lens = list(p.req), list(p.lens)
    p.req[6] = p.R
    p.lens[4] = p.max_pages * 16 + 1
    o, ls = p.call()
    bad = torch.tensor([False] * 4 + [True, False, True, False], device="cuda")
    assert bool(torch.isnan(o[bad]).all()) and bool(torch.isnan(ls[bad]).all())
    assert float((o[~bad] - want[~bad]).abs().max()) < 2.0 ** -18


def test_attention_shared_starts_without_order():
    """Groups that overlap, run backwards or past the rows: no row of another group's business, nothing out of range."""
    p = Shared([([40, 41, 42, 43], 40), ([50, 51], 50), ([9], 9)], 8, 2, 64, 16, "f16", "f16")
    guard = torch.full((len(p.lens) + 2, 8, 64), 5.0, device="cuda", dtype=p.dt)
    for starts in ([4, 2, 0, 7], [0, 9, 2, 100], [-5, 3, 3, 2], [7, 7, 7, 7], [0, 0, 0, -1], [2 ** 31 - 1] * 4, [-2 ** 31] * 4):
        p.call(starts=starts, out=guard[1:-1])
        torch.cuda.synchronize()
        assert bool((guard[0] == 5).all()) and bool((guard[-1] == 5).all())
    for starts in ([7, 7, 7, 7], [-9, -3, -2, 0]):
        p.check(*p.call(starts=starts))


def test_attention_shared_strided_rows():
    p = Shared([([130, 140, 129, 128], 128), ([33], 0)], 8, 2, 64, 16, "bf16", "bf16")
    want, lw = p.call()
    B = len(p.lens)
    for off, qs, os_, ts in ((1, 521, 515, 0), (0, 0, 0, 0), (8, 520, 528, 1), (3, 512 + 3, 512, 5)):
        mem = torch.full((B * 600,), math.nan, device="cuda", dtype=p.dt)
        q = torch.as_strided(mem, (B, 8, 64), (qs or 512, 64, 1), off)
        q.copy_(p.q)
        omem = torch.full((B * 600,), 5.0, device="cuda", dtype=p.dt)
        out = torch.as_strided(omem, (B, 8, 64), (os_ or 512, 64, 1), off)
        table = p.table
        if ts:
            wide = torch.full((p.R, p.max_pages + ts), 10 ** 9, dtype=torch.int32, device="cuda")
            wide[:, :p.max_pages] = table
            p.table = wide
        o, ls = p.call(q=q, out=out, q_stride=qs, out_stride=os_, table_stride=p.max_pages + ts if ts else 0)
        p.table = table
        assert torch.equal(o, want) and torch.equal(ls, lw)
        out.fill_(5.0)
        assert bool((omem == 5).all())


@pytest.mark.parametrize("size", [1e-30, 1e-10, 1e10, 1e30, 3e38])
@pytest.mark.parametrize("cache", ["f16", "bf16"])
def test_attention_shared_range_of_q(size, cache):
    """fp32 rows of any magnitude: the scale of a row is taken out before it becomes 16-bit terms."""
    p = Shared([([200, 210, 199], 190)], 4, 2, 64, 16, "f32", cache)
    p.q = p.q / p.q.abs().amax(2, keepdim=True) * size
    scale = 1.0 / size if size < 1e37 else 2.0 ** -126
    p.check(*p.call(scale=scale), scale=scale)


def test_attention_shared_infinite_scores():
    """Keys that make scores -inf have weight zero; a row whose scores are all -inf is like one that sees nothing."""
    p = Shared([([70, 75], 64), ([20, 20], 20)], 4, 2, 64, 16, "f32", "f16")
    p.q = p.q.abs()
    for b, pos in ((0, 3), (0, 66), (1, 70)):
        p.kc[int(p.table[b, pos // 16]), pos % 16] = -math.inf
    for pos in range(20):
        p.kc[int(p.table[2, pos // 16]), pos % 16] = -math.inf
    o, ls = p.call()
    a, la = Paged.call(p)
    assert bool((o[2:] == 0).all()) and bool((ls[2:] == -math.inf).all())
    assert bool(torch.isfinite(o[:2]).all())
    assert float((o[:2] - a[:2]).norm() / a[:2].norm()) < 2.0 ** -19 and float((ls[:2] - la[:2]).abs().max()) < 2.0 ** -17


def test_attention_shared_streams_and_graph():
    """Two calls at once with scratch of their own; one captured and replayed as lengths, groups, tables and rows change."""
    ps = [Shared([([500 + i, 510, 530], 500), ([77 + i], 50)], 16, 4, 64, 16, "bf16", "bf16", seed=i) for i in range(2)]
    want = [[t.clone() for t in p.call()] for p in ps]
    torch.cuda.synchronize()
    streams, outs = [torch.cuda.Stream() for _ in ps], [[] for _ in ps]
    for _ in range(10):
        for p, s, o in zip(ps, streams, outs):
            with torch.cuda.stream(s):
                o.append(p.call(scratch=p.scratch))
    torch.cuda.synchronize()
    for w, o in zip(want, outs):
        for got in o:
            assert torch.equal(got[0], w[0]) and torch.equal(got[1], w[1])
    p = Shared([([400, 410, 420, 401], 400), ([30, 31], 16)], 16, 4, 64, 16, "bf16", "bf16", seed=3)
    out, ls = p.call()
    lens, starts, prefix = p.lens_d, p.starts_d, p.prefix_d
    kv = b2.paged_kv(p.kc.data_ptr(), p.vc.data_ptr(), p.cid, p.total, 16, 4, 64)
    o = b2.paged_attn_opts(p.tid, 16, p.R, p.max_pages)

    def call():
        b2.attention_shared(kv, o, p.q.data_ptr(), p.table.data_ptr(), lens.data_ptr(), p.req_d.data_ptr(), 6, starts.data_ptr(),
                            prefix.data_ptr(), 2, out.data_ptr(), ls.data_ptr(), p.scratch.data_ptr(), stream())
    call()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        call()
    for ln, st, pre in (([400, 410, 420, 401, 30, 31], [0, 4, 6], [400, 16]), ([1, 0, 5, 7, 30, 2], [0, 4, 6], [1, 0]),
                        ([400, 400, 400, 400, 30, 30], [0, 4, 4], [384, 0]), ([0] * 6, [0, 4, 6], [400, 16])):
        lens.copy_(i32(ln))
        starts.copy_(i32(st))
        prefix.copy_(i32(pre))
        p.lens = ln
        out.fill_(5)
        ls.fill_(5)
        g.replay()
        p.check(out, ls)


def test_attention_shared_same_bits_again():
    p = Shared([([3000 + i for i in range(30)], 3000), ([500, 600], 500)], 16, 2, 128, 16, "f32", "bf16")
    a, la = p.call()
    for _ in range(3):
        o, ls = p.call()
        assert torch.equal(a, o) and torch.equal(la, ls)


def test_attention_shared_offsets_past_32_bits():
    """Pages that lie 6 GB behind the cache's start."""
    nkv, hd, P = 8, 128, 64
    page = P * nkv * hd
    far = (6 << 30) // (2 * page)
    mem = torch.zeros(2, far + 3, page, dtype=torch.bfloat16, device="cuda")
    p = Shared([([150, 170, 180], 128)], 32, nkv, hd, P, "bf16", "bf16")
    want, lw = p.call()
    k, v = (m.view(far + 3, P, nkv, hd) for m in mem)
    table = torch.full_like(p.table, -1)
    used = torch.unique(p.table[p.table >= 0]).tolist()
    place = [far + 2, far, far - 3, far + 1, far - 1, far - 2, 0, 1, 2]
    for i, pg in enumerate(used):
        k[place[i]], v[place[i]] = p.kc[pg], p.vc[pg]
        table[p.table == pg] = place[i]
    p.kc, p.vc, p.table, p.total = k, v, table, far + 3
    o, ls = p.call()
    assert torch.equal(o, want) and torch.equal(ls, lw)


def test_attention_shared_behind_its_plan():
    """b2_page_plan's starts and lengths as the groups: prompts and single tokens of one step, padding rows behind them."""
    g = np.random.default_rng(5)
    cached, fresh = np.array([0, 200, 37, 0, 513]), np.array([150, 1, 40, 0, 1])
    P, nh, nkv, hd, cap, R = 16, 8, 2, 64, 200, 5
    mp = 100
    n_pages = 120
    ids = g.permutation(n_pages).astype(np.int32)
    table, at = np.full((R, mp), -1, np.int32), 0
    for r in range(R):
        n = -(-int(cached[r]) // P)
        table[r, :n] = ids[at:at + n]
        at += n
    td, cd, fd, free, nf = i32(table), i32(cached), i32(fresh), i32(ids[at:]), i32([n_pages - at])
    new = lambda n, t=torch.int32: torch.empty(n, dtype=t, device="cuda")  # noqa: E731
    lens, starts, slots, pos, req, info = new(R), new(R + 1), new(cap, torch.int64), new(cap), new(cap), new(4)
    gen = torch.Generator(device="cuda").manual_seed(1)
    kc, vc = torch.randn(2, n_pages, P, nkv, hd, device="cuda", generator=gen).to(torch.bfloat16)
    q = torch.randn(cap, nh, hd, device="cuda", generator=gen).to(torch.bfloat16)
    out, ls = torch.full((cap, nh, hd), 5.0, device="cuda", dtype=torch.bfloat16), torch.full((cap, nh), 5.0, device="cuda")
    kv = b2.paged_kv(kc.data_ptr(), vc.data_ptr(), b2.BF16, n_pages, P, nkv, hd)
    o = b2.paged_attn_opts(b2.BF16, nh, R, mp, len_add=1)
    scratch = torch.empty(b2.attention_shared_scratch_bytes(cap, nh, nkv, hd), dtype=torch.uint8, device="cuda")

    def step():
        b2.page_plan(cd.data_ptr(), fd.data_ptr(), R, P, free.data_ptr(), nf.data_ptr(), td.data_ptr(), mp, mp, lens.data_ptr(),
                     starts.data_ptr(), slots.data_ptr(), pos.data_ptr(), req.data_ptr(), cap, info.data_ptr(), stream())
        b2.attention_shared(kv, o, q.data_ptr(), td.data_ptr(), pos.data_ptr(), req.data_ptr(), cap, starts.data_ptr(),
                            lens.data_ptr(), R, out.data_ptr(), ls.data_ptr(), scratch.data_ptr(), stream())
    step()
    assert info.tolist()[0] == 0
    T = int(fresh.sum())
    vmax = float(vc.float().abs().max())
    want, lse, to, tl = attend64(q, kc, vc, td, [x + 1 for x in pos.tolist()], req.tolist(), P, 0, hd ** -0.5, 0.0, None)
    to = to + half_step(torch.bfloat16) * vmax  # (probabilities of one term)
    assert_within(out, want, to[..., None].expand_as(want), torch.bfloat16)
    assert bool((out[T:] == 0).all()) and bool((ls[T:] == -math.inf).all())
    assert float((out[:T].double() - want[:T]).norm() / want[:T].norm()) <= half_step(torch.bfloat16)
