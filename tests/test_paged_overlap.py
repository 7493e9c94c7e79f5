"""Arguments of the paged serving operators that share memory.

The entry points look at addresses and sizes before they launch anything:
tests/overlap_check.cpp compiles that arithmetic (csrc/overlap.h) as plain C++,
so that it is checked without a device; the refusals themselves are called on
one where they come behind the pointers' own checks."""
import os
import subprocess

import pytest

import b2decode as b2

HERE = os.path.dirname(os.path.abspath(__file__))
ARRAYS = ("cached", "fresh", "free_pages", "n_free", "table", "lens", "starts", "slots", "positions", "token_req", "info")
SIZES = ("n_req", "max_pages", "table_stride", "max_tokens")


@pytest.fixture(scope="module")
def check(tmp_path_factory):
    exe = str(tmp_path_factory.mktemp("overlap") / "overlap_check")
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-I/usr/local/cuda/include", "-o", exe,
                    os.path.join(HERE, "overlap_check.cpp")], check=True)
    return exe


def plan(check, **kw):
    args = [str(kw[n]) for n in ARRAYS + SIZES]
    return subprocess.run([check, *args], check=True, capture_output=True, text=True).stdout.strip()


def packed(n_req, max_pages, stride, max_tokens, at=1 << 32):
    """The arrays back to back, none sharing a byte with the next."""
    size = dict(cached=4 * n_req, fresh=4 * n_req, free_pages=4, n_free=4, table=4 * ((n_req - 1) * stride + max_pages),
                lens=4 * n_req, starts=4 * (n_req + 1), slots=8 * max_tokens, positions=4 * max_tokens,
                token_req=4 * max_tokens, info=16)
    kw = dict(n_req=n_req, max_pages=max_pages, table_stride=stride, max_tokens=max_tokens)
    for n in ARRAYS:
        kw[n] = at
        at += size[n]
    return kw, size


def test_regions_meet(check):
    out = subprocess.run([check, "meet"], capture_output=True, text=True)
    assert out.returncode == 0 and out.stdout.startswith("0 of"), out.stdout


@pytest.mark.parametrize("shape", [(1, 1, 1, 1), (4, 8, 8, 64), (16384, 1000, 1003, 1 << 20)])
def test_neighbours_are_accepted(check, shape):
    kw, _ = packed(*shape)
    assert plan(check, **kw) == "ok"
    assert plan(check, **{**kw, "fresh": kw["cached"], "n_free": kw["cached"]}) == "ok"  # read alone


@pytest.mark.parametrize("out", ["table", "lens", "starts", "slots", "positions", "token_req", "info"])
@pytest.mark.parametrize("inp", ["cached", "fresh", "free_pages", "n_free", "table"])
def test_an_output_on_an_input_is_refused(check, out, inp):
    """The same start, and one word shared at either end."""
    if out == inp:
        return
    kw, size = packed(5, 7, 9, 30)
    for at in (kw[inp], kw[inp] + size[inp] - 4, kw[inp] - size[out] + 4):
        said = plan(check, **{**kw, out: at})
        assert " overlaps " in said and out in said, said


def test_between_the_rows_of_a_table(check):
    kw, _ = packed(5, 7, 16, 30)
    row = 4 * 16
    assert plan(check, **{**kw, "info": kw["table"] + 2 * row + 4 * 7}) == "ok"
    assert plan(check, **{**kw, "info": kw["table"] + 2 * row + 4 * 6}) == "info overlaps table"
    assert plan(check, **{**kw, "info": kw["table"] + 2 * row + 4 * 13}) == "info overlaps table"


PTR = 1 << 20  # an address that no refused call reads


def append(**kw):
    a = dict(k_ptr=PTR, v_ptr=PTR + (1 << 30), dtype=b2.F16, n_pages=4, page_size=16, nkv=2, hd=64)
    a.update(kw)
    kv = b2.paged_kv(**a)
    rows = b2.rope_rows(b2.F16, 4, kv.nkv, kv.hd, kv.hd)
    with pytest.raises(b2.B2Error) as e:
        b2.rope_append(rows, kv, PTR, PTR, PTR, 3, PTR, PTR, PTR, PTR)
    return "place elements on one another" in str(e.value)


E = 16 * 2 * 64  # elements of a dense page


@pytest.mark.parametrize("change", [
    dict(v_ptr=PTR),  # k and v the same memory
    dict(v_ptr=PTR + 2 * E),  # v one page into k's four
    dict(v_ptr=PTR + 16),
    dict(page_stride=E, pos_stride=128, head_stride=0),  # heads on one another
    dict(page_stride=E, pos_stride=128, head_stride=56),
    dict(page_stride=E, pos_stride=120, head_stride=64),  # positions
    dict(page_stride=E - 8, pos_stride=128, head_stride=64),  # pages
    dict(page_stride=0, pos_stride=128, head_stride=64),
    dict(page_stride=E, pos_stride=64, head_stride=64 * 15),  # heads in a page of 15 positions
    dict(page_stride=E, pos_stride=128, head_stride=64, v_ptr=PTR + 2 * E),  # k and v alternate by pages of a stride for one
])
def test_cache_places_on_one_another_are_refused(built_lib, change):
    assert append(**change)


@pytest.mark.parametrize("change", [
    dict(), dict(v_ptr=PTR + 4 * 2 * E), dict(k_ptr=PTR + 4 * 2 * E, v_ptr=PTR),
    dict(page_stride=E, pos_stride=64, head_stride=64 * 16),  # head-major
    dict(page_stride=2 * E, pos_stride=128, head_stride=64, v_ptr=PTR + 2 * E),  # k and v of a page together
    dict(page_stride=2 * E, pos_stride=256, head_stride=64, v_ptr=PTR + 2 * 128),  # of a position
    dict(page_stride=2 * E, pos_stride=256, head_stride=128, v_ptr=PTR + 2 * 64),  # of a head
    dict(page_stride=128, pos_stride=512, head_stride=64),  # pages inside positions
    dict(n_pages=1, page_stride=8, pos_stride=128, head_stride=64), dict(nkv=1, head_stride=8, pos_stride=64, page_stride=1024),
    dict(n_pages=1, nkv=1, page_size=1, page_stride=8, v_ptr=PTR + 128),
])
def test_cache_layouts_that_stay_accepted(built_lib, change):
    """(They fail later: the addresses are no memory.)"""
    assert not append(**change)


@pytest.mark.gpu
@pytest.mark.parametrize("out,inp", [("lens", "cached"), ("lens", "fresh"), ("starts", "cached"), ("info", "n_free"),
                                     ("positions", "table"), ("table", "free_pages")])
def test_page_plan_refuses_shared_memory(out, inp):
    torch = pytest.importorskip("torch")
    a = {n: torch.zeros(64, dtype=torch.int64, device="cuda") for n in ARRAYS}
    a[out] = a[inp]
    with pytest.raises(b2.B2Error, match="b2_page_plan: .* overlaps ") as e:
        b2.page_plan(a["cached"].data_ptr(), a["fresh"].data_ptr(), 4, 16, a["free_pages"].data_ptr(),
                     a["n_free"].data_ptr(), a["table"].data_ptr(), 8, 8, a["lens"].data_ptr(), a["starts"].data_ptr(),
                     a["slots"].data_ptr(), a["positions"].data_ptr(), a["token_req"].data_ptr(), 16,
                     a["info"].data_ptr())
    assert e.value.code == -8
    assert all(bool((t == 0).all()) for t in a.values())
