"""b2_matvec from several host threads at once."""
import threading

import pytest

import b2decode as b2

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


@pytest.mark.parametrize("qtype,block", [(8, 34), (2, 18)])
def test_threads_of_different_widths(qtype, block):
    """Rows of different widths want different amounts of shared memory: no call makes another's launch fail, and the
    results are those of one thread."""
    rows, calls, codes = 64, [], []
    g = torch.Generator(device="cuda").manual_seed(qtype)
    for cols in (256, 8192, 16384, 4096):
        w = torch.randint(0, 256, (rows, cols // 32, block), dtype=torch.uint8, device="cuda", generator=g)
        w[:, :, 0], w[:, :, 1] = 0, 0x28  # the blocks' scales: 2^-5 as fp16
        x, y = torch.randn(cols, device="cuda", generator=g), torch.zeros(rows, device="cuda")
        b2.matvec(qtype, w.data_ptr(), x.data_ptr(), y.data_ptr(), rows, cols, torch.cuda.current_stream().cuda_stream)
        calls.append((w, x, y.clone(), torch.zeros_like(y), cols))
    torch.cuda.synchronize()
    start = threading.Barrier(len(calls))

    def run(w, x, _, y, cols):
        st = torch.cuda.Stream()
        a = (qtype, w.data_ptr(), x.data_ptr(), y.data_ptr(), rows, cols, st.cuda_stream)
        f = b2.lib().b2_matvec
        start.wait()
        for _ in range(8):
            codes.extend({f(*a) for _ in range(500)})
            st.synchronize()
    threads = [threading.Thread(target=run, args=c) for c in calls]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert set(codes) == {0}
    for _, _, want, y, _ in calls:
        assert torch.equal(y, want)
