"""The beam search's operators where two candidates, two threads or two sizes meet
at a border."""
import pytest

from test_gpu_beam import Select
from test_gpu_paged import DT

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
