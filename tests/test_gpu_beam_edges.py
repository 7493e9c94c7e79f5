"""The beam search's operators where two candidates, two threads or two sizes meet
at a border."""
import math
import threading

import pytest

import b2decode as b2
from test_gpu_beam import Select
from test_gpu_paged import DT, E32, i32, stream

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("W,k", [(2, 1), (2, 3), (4, 1), (4, 3), (4, 5), (8, 7), (3, 2)])
def test_doubled_logits_at_the_last_place(dtype, W, k):
    """Every logit stands twice in its row and the beams' best candidates are within 2e-7 of one another, so places
    k - 1 and k are one beam's and the candidate that rivals them comes behind: the choice is that of 64 bits."""
    G, n = 200, 20000
    g = torch.Generator(device="cuda").manual_seed(W * 10 + k)
    x = 2.5 * torch.randn(G * W, n // 2, device="cuda", generator=g)
    x = torch.cat([x, x], 1)[:, torch.randperm(n, device="cuda", generator=g)].to(DT[dtype][0]).contiguous()
    d = x.double()
    best = d.amax(1) - torch.logsumexp(d, 1)
    near = 2e-7 * torch.rand(G * W, device="cuda", dtype=torch.float64, generator=g)
    Select(x, n, G, W, k, -1, (near - 1.0 - best).float()).call().check()


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("pad", [0, 1])
def test_scores_of_a_sure_token(dtype, pad):
    """One logit far above the others, which lie within 1 of 0: log p = -log(1 + r) with r = sum e^(x - m).  Every
    term of r is off by at most 2 steps in its exponential and in each factor that raises its reference (3 2^-22),
    and by 2.25 half steps of |d| < 30 in d log2(e) (2^-17.9): 2^-17 in all.  The up to 31 terms that are summed
    with the largest, some 32 e^2 / n of r at most, may be lost there.  The score is rounded once."""
    n, G = 65536, 12
    g = torch.Generator(device="cuda").manual_seed(3)
    x = (2 * torch.rand(G, n + pad, device="cuda", generator=g) - 1).to(DT[dtype][0])
    at = torch.randint(1, n, (G, 1), device="cuda", generator=g)
    x.scatter_(1, at, torch.linspace(14, 28, G, device="cuda")[:, None].to(x.dtype))
    lp = torch.log_softmax(x[:, :n].double(), 1)
    d = (x[:, :n].double() - x[:, :n].double().amax(1, keepdim=True)).scatter(1, at, -math.inf)
    want = -torch.log1p(torch.exp(d).sum(1))
    assert float((want - lp.gather(1, at)[:, 0]).abs().max()) < 1e-12
    s = Select(x, n, G, 1, 1, 0).call()
    s.check()
    tol = want.abs() * (2.0 ** -17 + 32 * math.e ** 2 / n + E32)
    err = (s.score[:G].double() - want).abs()
    assert bool((err <= tol).all()), (err / want.abs()).tolist()
    # the same token as the end token
    for i in range(G):
        e = Select(x[i:i + 1], n, 1, 1, 1, int(at[i])).call()
        assert abs(float(e.eos_score[0]) - float(want[i])) <= float(tol[i])


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_one_log_z_of_a_row(dtype):
    """Beams with nearly the same logits in other places come close, so their log Z are taken in 64 bits; the end
    token's score has the same log Z: the value in 64 bits (whose sums are off by some 1e-13), rounded once.

    Which beams: e^d of the end token is 1, the others weigh 0.16 together with |d| near 13, so fp32 log Z are off by
    0.16 (13 * 2.25 half steps + 3 2^-22) + 8 half steps < 2^-20.  Neighbours of two beams within 2^-18 are then
    within 2^-18 + 2^-19 for the kernel, which settles what is within 2^-17."""
    G, W, n, eos = 8, 8, 50000, 77
    g = torch.Generator(device="cuda").manual_seed(5)
    x = torch.randn(G, 1, n, device="cuda", generator=g).expand(G, W, n).contiguous()
    for r in x.view(-1, n):
        r.copy_(r[torch.randperm(n, device="cuda", generator=g)])
    x[:, :, eos] = 13.0
    x = x.view(G * W, n).to(DT[dtype][0])
    s = Select(x, n, G, W, 4 * W, eos).call()
    lp = torch.log_softmax(x.double(), 1)
    want = lp[:, eos].clone()
    score = lp[s.parent[:-1].long(), s.token[:-1].long()]
    lp[:, eos] = -math.inf
    val, at = torch.sort(lp.view(G, W * n), dim=1, descending=True, stable=True)
    row = (torch.arange(G, device="cuda")[:, None] * W + at // n)[:, :4 * W]
    near = (row[:, 1:] != row[:, :-1]) & (val[:, :4 * W - 1] - val[:, 1:4 * W] < 2.0 ** -18)
    settled = torch.zeros(G * W, dtype=torch.bool, device="cuda")
    settled[row[:, 1:][near]] = True
    settled[row[:, :-1][near]] = True
    assert int(settled.sum()) > G * W // 2
    err = (s.eos_score[:-1].double() - want).abs()
    assert bool((err <= E32 * want.abs() + 1e-12)[settled].all())
    err = (s.score[:-1].double() - score).abs()
    assert bool((err <= E32 * score.abs() + 1e-12)[settled[s.parent[:-1].long()]].all())


def test_threads_of_different_widths():
    """Threads whose requests want different amounts of shared memory, past what a launch may ask for as it is: no call
    makes another's launch fail."""
    n, codes = 200, []
    x = torch.randn(64, n, device="cuda", generator=torch.Generator(device="cuda").manual_seed(1))
    calls = [Select(x[:w], n, 1, w, 64) for w in (64, 48, 64, 48)]
    torch.cuda.synchronize()
    start = threading.Barrier(len(calls))

    def run(s):
        st = torch.cuda.Stream()
        f = b2.lib().b2_beam_select
        a = (s.x.data_ptr(), b2.F32, n, 1, s.W, n, None, 64, -1, s.parent.data_ptr(), s.token.data_ptr(), s.score.data_ptr(), None,
             s.scratch.data_ptr(), st.cuda_stream)
        start.wait()
        for _ in range(8):
            codes.extend({f(*a) for _ in range(500)})
            st.synchronize()
    threads = [threading.Thread(target=run, args=(s,)) for s in calls]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert set(codes) == {0}
    for s in calls:
        s.check()


def test_pages_up_to_2_31():
    """A pool of 2^31 - 1 pages and rows of as many entries, few of them in use: counted, listed, forked, compacted."""
    torch.cuda.empty_cache()
    N = 2 ** 31 - 1
    big = lambda n=N: torch.empty(n, dtype=torch.int32, device="cuda")  # noqa: E731
    table, refs, free, n_free, lens = big(), big(), big(), i32([-9]), i32([70])
    used = [0, N - 2, 5, 2 ** 30, N - 1]
    table[:6] = i32(used + [77])
    refs.fill_(-9)
    scratch = torch.empty(max(b2.page_pool_scratch_bytes(N), b2.page_compact_scratch_bytes(N)), dtype=torch.uint8, device="cuda")

    def pool(t):
        b2.page_pool(t.data_ptr(), N, lens.data_ptr(), 1, 16, N, refs.data_ptr(), N, free.data_ptr(), n_free.data_ptr(),
                     scratch.data_ptr(), stream())
        assert int(n_free) == N - 5
    pool(table)
    assert int(torch.count_nonzero(refs)) == 5 and refs[used].tolist() == [1] * 5
    gaps = torch.tensor(sorted(used), device="cuda") - torch.arange(5, device="cuda")
    for at in range(0, N - 5, 1 << 28):  # free[i] = i and the pages in use before it
        i = torch.arange(at, min(at + (1 << 28), N - 5), device="cuda")
        assert torch.equal(free[at:at + len(i)].long(), i + torch.bucketize(i, gaps, right=True))
    parent, new, new_lens, pairs, info = i32([0]), big(), i32([-9, -9]), torch.full((8, 3), -9, dtype=torch.int32, device="cuda"), i32([-9] * 4)
    b2.page_fork(parent.data_ptr(), 1, table.data_ptr(), N, lens.data_ptr(), 1, 16, refs.data_ptr(), N, free.data_ptr(),
                 n_free.data_ptr(), new.data_ptr(), N, N, new_lens.data_ptr(), pairs.data_ptr(), info.data_ptr(), stream())
    assert info.tolist() == [0, 0, 0, 0] and new_lens.tolist() == [70, -9] and new[:5].tolist() == used
    b2.page_compact(new.data_ptr(), N, lens.data_ptr(), 1, 16, N, refs.data_ptr(), N, pairs.data_ptr(), 7, info.data_ptr(),
                    scratch.data_ptr(), stream())
    assert info.tolist() == [0, 4, 5, 5] and new[:5].tolist() == [0, 2, 4, 3, 1]
    assert pairs.tolist() == [[N - 1, 1, 16], [N - 2, 2, 16], [2 ** 30, 3, 16], [5, 4, 16]] + [[-9] * 3] * 4
    pool(new)
    assert refs[:6].tolist() == [1] * 5 + [0] and free[:3].tolist() == [5, 6, 7]
    del table, refs, free, new, scratch
    torch.cuda.empty_cache()
