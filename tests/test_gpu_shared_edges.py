"""Attention of shared prefixes where its weights, lengths, prefixes and repairs
are at the ends of their ranges."""
import math

import pytest

from test_gpu_paged import DT
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
