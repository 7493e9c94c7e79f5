"""Attention of shared prefixes where its weights, lengths, prefixes and repairs
are at the ends of their ranges."""
import math

import pytest

import b2decode as b2
from test_gpu_paged import DT, assert_within, attend64, i32, stream
from test_gpu_shared import Shared

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("one", [False, True])
@pytest.mark.parametrize("hd", [64, 128])
def test_constant_values_come_out_as_they_are(dtype, one, hd):
    """Weights that add up to one: of values that are 1.5 throughout, 1.5.  One position in 16 has the largest
    score, the others a weight half a step of the type above 1/2, so weights of one 16-bit term are all off to the
    same side: by 15/17 of a half step in the sum, which in 1.5 is 1.3 half steps and shows.  Two terms leave 2^-16
    of it."""
    eps = torch.finfo(DT[dtype][0]).eps
    lens = [1024 + 16 * i for i in range(40)]
    p = Shared([(lens, max(lens) if one else 1024), ([333 + i for i in range(50)], 382 if one else 333)], 16, 2, hd, 16, dtype, dtype,
               one=one)
    p.kc.zero_()
    p.kc[:, 0, :, 0] = 1
    p.vc.fill_(1.5)
    p.q.zero_()
    p.q[..., 0] = 1
    out, _ = p.call(scale=-math.log(0.5 * (1 + eps / 2)))
    assert bool((out == 1.5).all()), out.unique().tolist()


@pytest.mark.parametrize("dtype,cache", [("f32", "f16"), ("bf16", "bf16")])
@pytest.mark.parametrize("prefix", [2 ** 31 - 1, 2 ** 31 - 2])
@pytest.mark.parametrize("groups", [[list(range(270, 310)), [40, 41], [700] * 3], [list(range(9000, 9030))]])
def test_prefix_of_everything(dtype, cache, prefix, groups):
    """A prefix past every length: all of it is shared, whether an item is written whole (many of them) or in pieces."""
    p = Shared([(ls, max(ls)) for ls in groups for _ in range(40 if len(groups) > 1 else 1)], 16, 2, 64, 16, dtype, cache, one=True)
    p.check(*p.call(prefix=[prefix] * len(p.prefix)))


@pytest.mark.parametrize("P", [8, 16, 24, 100])
@pytest.mark.parametrize("dtype,cache", [("f32", "f16"), ("bf16", "bf16")])
def test_missing_page_at_every_place(P, dtype, cache):
    """Group i's page i does not exist, in whichever tile and part of it that is, by boxes or row by row: its rows are
    NaN, and all of a call in which it is whole is as it was."""
    places = 640 // P
    p = Shared([([640, 641, 655], 640) for _ in range(places)], 8, 2, 64, P, dtype, cache)
    want = p.call()[0].clone()
    keep = p.table.clone()
    for r in range(len(p.lens)):
        p.table[r, r // 3] = -1 if r % 2 else p.total
    for _ in range(5):
        out, ls = p.call()
        assert bool(torch.isnan(out).all()) and bool(torch.isnan(ls).all())
    p.table = keep
    assert torch.equal(p.call()[0], want)


@pytest.mark.parametrize("size", [1.0, 1e30, 3e38])
@pytest.mark.parametrize("cache", ["f16", "bf16"])
def test_large_queries_beside_infinite_values(size, cache):
    """fp32 rows of any magnitude in a group where another row sees an infinite value: those that do not see it get
    what they get without it."""
    p = Shared([([100, 128, 200, 90, 330], 330)], 8, 2, 64, 16, "f32", cache, one=True)
    p.q = p.q / p.q.abs().amax(2, keepdim=True) * size
    scale = 0.125 if size == 1.0 else 1.0 / size if size < 1e37 else 2.0 ** -126
    p.vc[int(p.table[0, 150 // 16]), 150 % 16] = math.inf
    out, ls = p.call(scale=scale)
    want, lse, to, tl = attend64(p.q, p.kc, p.vc, p.table, p.lens, p.req, 16, 0, scale, 0.0, None)
    for b in (0, 1, 3):
        assert_within(out[b], want[b], to[b][:, None].expand_as(want[b]), torch.float32)
        assert bool(((ls[b].double() - lse[b]).abs() <= tl[b]).all())
    assert bool((out[[2, 4]] == math.inf).all())


@pytest.mark.parametrize("dtype,cache", [("f32", "f16"), ("bf16", "bf16")])
@pytest.mark.parametrize("prefix", [2 ** 31 - 1, 100])
def test_longest_rows(dtype, cache, prefix):
    """Two rows of 2^31 - 64 positions and a few less, every page of theirs the same one; their positions together,
    or each row's own.  A position j of the page weighs as often as it is seen, c_j, so out = sum c_j e^s_j v_j / sum
    c_j e^s_j and lse = log of that sum.  2^24 tiles go to 148 shares, and a share's sums run over 2^17 tiles (twice
    as many where there are two rows) in fp32: each addition rounds by half a step, 2^18 2^-24 = 2^-6 of the sum
    at worst, and twice that in the quotient; the join and the rounding of out are far below."""
    P, nh, hd = 65536, 8, 64
    dt, tid = DT[dtype]
    ct, cid = DT[cache]
    g = torch.Generator(device="cuda").manual_seed(1)
    kc = torch.randn(1, P, 1, hd, device="cuda", generator=g).to(ct)
    vc = (1 + torch.randn(1, P, 1, hd, device="cuda", generator=g)).to(ct)
    q = torch.randn(2, nh, hd, device="cuda", generator=g).to(dt)
    lens, pages = [2 ** 31 - 64, 2 ** 31 - 1000], 2 ** 31 // P
    table = torch.zeros(2, pages, dtype=torch.int32, device="cuda")
    out, lse = torch.full((2, nh, hd), 5.0, device="cuda", dtype=dt), torch.full((2, nh), 5.0, device="cuda")
    scratch = torch.empty(b2.attention_shared_scratch_bytes(2, nh, 1, hd), dtype=torch.uint8, device="cuda")
    kv = b2.paged_kv(kc.data_ptr(), vc.data_ptr(), cid, 1, P, 1, hd)
    opts = b2.paged_attn_opts(tid, nh, 2, pages)
    ln, starts, pre = i32(lens), i32([0, 2]), i32([prefix])
    b2.attention_shared(kv, opts, q.data_ptr(), table.data_ptr(), ln.data_ptr(), 0, 2, starts.data_ptr(), pre.data_ptr(), 1,
                        out.data_ptr(), lse.data_ptr(), scratch.data_ptr(), stream())
    k, v = kc[0, :, 0].double(), vc[0, :, 0].double()
    for b, n in enumerate(lens):
        c = n // P + (torch.arange(P, device="cuda") < n % P).double()
        s = q[b].double() @ k.T / 8 + torch.log(c)
        want = torch.softmax(s, 1) @ v
        tol = 2.0 ** -5 * v.abs().max()
        assert_within(out[b], want, tol.expand_as(want), dt)
        assert bool(((lse[b].double() - torch.logsumexp(s, 1)).abs() <= 2.0 ** -5).all())
