"""The operators of a beam search over a paged cache without a GPU: every
refusal of their entry points comes before the first CUDA call, so it is the
same with and without a device."""
import math

import pytest

import b2decode as b2

# addresses that no refused call reads, far enough apart for every size below
A = [(i + 1) << 32 for i in range(16)]
P = A[0]


def refused(code, text, fn, *args, **kw):
    with pytest.raises(b2.B2Error) as e:
        fn(*args, **kw)
    assert e.value.code == code and text in str(e.value), str(e.value)


SELECT = dict(logits=A[0], dtype=b2.F32, n=100, n_groups=3, width=4, ld=100, scores=A[1], k=4, eos=-1, parent=A[2],
              token=A[3], score=A[4], eos_score=A[5], scratch=A[6])


@pytest.mark.parametrize("change,code", [
    ({"dtype": 8}, -3), ({"n": 0}, -8), ({"n": (1 << 30) + 1, "ld": 1 << 31}, -8), ({"ld": 99}, -8), ({"n_groups": 0}, -8),
    ({"width": 0}, -8), ({"width": 65}, -8), ({"n_groups": 1 << 25, "width": 8}, -8), ({"k": 0}, -8), ({"k": 65}, -8),
    ({"k": 11, "n": 10}, -8), ({"eos": 100}, -8)]
    + [({k: 0}, -8) for k in ("logits", "parent", "token", "score", "scratch")])
def test_beam_select_refusals(built_lib, change, code):
    refused(code, "b2_beam_select", b2.beam_select, **{**SELECT, **change})


@pytest.mark.parametrize("name", ["logits", "scores", "parent", "token", "score", "eos_score", "scratch"])
def test_beam_select_misaligned(built_lib, name):
    refused(-8, "aligned", b2.beam_select, **{**SELECT, name: P + 1})
    refused(-8, "aligned", b2.beam_select, **{**SELECT, "scratch": P + 8})


@pytest.mark.parametrize("out", ["parent", "token", "score", "eos_score", "scratch"])
def test_beam_select_overlaps(built_lib, out):
    a = {**SELECT, "eos": 7}
    refused(-8, "overlaps", b2.beam_select, **{**a, out: a["scores"]})
    refused(-8, "overlaps", b2.beam_select, **{**a, out: a["logits"] + 4 * 99 + 4 * 100 * 11 - 12})
    other = "token" if out != "token" else "score"
    refused(-8, "overlaps", b2.beam_select, **{**a, out: a[other]})


def test_scratch_refusals(built_lib):
    for a in ((0, 1, 1, 1), (9, 0, 1, 1), (9, 1, 65, 1), (9, 1, 1, 65), (9, 1 << 25, 8, 1)):
        refused(-8, "scratch", b2.beam_select_scratch_bytes, *a)
    refused(-8, "scratch", b2.page_pool_scratch_bytes, 0)
    refused(-8, "scratch", b2.page_compact_scratch_bytes, -1)
    for a in ((0, 4, 2, 64), (4, 3, 2, 64), (4, 4, 0, 64), (4, 4, 2, 512)):
        refused(-8, "scratch", b2.attention_shared_scratch_bytes, *a)


REORDER = dict(src=A[0], n_src=3, src_stride=10, dst=A[1], n_dst=4, dst_stride=10, row_words=10, parent=A[2], lens=A[3],
               token=A[4], new_lens=A[5])


@pytest.mark.parametrize("change", [{"n_src": 0}, {"n_dst": 0}, {"row_words": 0}, {"src_stride": 9}, {"dst_stride": 9},
                                    {"src": 0}, {"dst": 0}, {"parent": 0}, {"src": P + 2}, {"new_lens": P + 1},
                                    {"dst": A[0] + 116}, {"dst": A[2]}, {"dst": A[3]}, {"dst": A[4]}, {"new_lens": A[0]},
                                    {"new_lens": A[3]}, {"new_lens": A[1] + 40}])
def test_beam_reorder_refusals(built_lib, change):
    refused(-8, "b2_beam_reorder", b2.beam_reorder, **{**REORDER, **change})


FORK = dict(parent=A[0], n_req=4, table=A[1], table_stride=8, lens=A[2], n_src=3, page_size=16, refs=A[3], n_pages=50,
            free_pages=A[4], n_free=A[5], new_table=A[6], new_stride=8, max_pages=8, new_lens=A[7], pairs=A[8], info=A[9])


@pytest.mark.parametrize("change", [
    {"n_req": 0}, {"n_req": 16385}, {"n_src": 0}, {"n_src": 16385}, {"page_size": 0}, {"n_pages": 0}, {"max_pages": 0},
    {"table_stride": 7}, {"new_stride": 7}]
    + [{k: 0} for k in ("parent", "table", "lens", "free_pages", "n_free", "new_table", "new_lens", "pairs", "info")]
    + [{k: P + 2} for k in ("parent", "table", "lens", "refs", "free_pages", "n_free", "new_table", "new_lens", "pairs", "info")]
    + [{"new_table": A[1] + 4 * 20}, {"new_table": A[0]}, {"new_lens": A[2]}, {"new_lens": A[0]}, {"pairs": A[3] + 196},
       {"info": A[5] - 12}, {"pairs": A[7]}, {"new_table": A[4]}])
def test_page_fork_refusals(built_lib, change):
    refused(-8, "b2_page_fork", b2.page_fork, **{**FORK, **change})


def kv(**kw):
    a = dict(k_ptr=A[0], v_ptr=A[1], dtype=b2.F16, n_pages=4, page_size=16, nkv=2, hd=64)
    a.update(kw)
    return b2.paged_kv(**a)


@pytest.mark.parametrize("change,code", [
    ({"k_ptr": 0}, -8), ({"dtype": b2.F32}, -3), ({"n_pages": 0}, -8), ({"hd": 60}, -8), ({"k_ptr": P + 8}, -8),
    ({"v_ptr": A[0] + 64}, -8), ({"page_stride": 1024, "pos_stride": 128, "head_stride": 64}, -8)])
def test_page_copy_cache_refusals(built_lib, change, code):
    refused(code, "b2_page_copy", b2.page_copy, kv(**change), 2, 1 << 20, A[3], A[4], 7)


@pytest.mark.parametrize("args", [
    (0, 1 << 20, A[3], A[4], 7), (2, -8, A[3], A[4], 7), (2, 1 << 20 | 4, A[3], A[4], 7), (2, 8192 - 8, A[3], A[4], 7),
    (2, 1 << 20, 0, A[4], 7), (2, 1 << 20, A[3], 0, 7), (2, 1 << 20, A[3], A[4], 0), (2, 1 << 20, A[3] + 2, A[4], 7)])
def test_page_copy_refusals(built_lib, args):
    refused(-8, "b2_page_copy", b2.page_copy, kv(), *args)


POOL = dict(table=A[0], table_stride=8, lens=A[1], n_req=4, page_size=16, max_pages=8, refs=A[2], n_pages=50,
            free_pages=A[3], n_free=A[4], scratch=A[5])


@pytest.mark.parametrize("change", [
    {"n_req": 0}, {"n_req": 16385}, {"page_size": 0}, {"n_pages": 0}, {"max_pages": 0}, {"table_stride": 7}]
    + [{k: 0} for k in ("table", "lens", "refs", "free_pages", "n_free", "scratch")]
    + [{k: P + 2} for k in ("table", "lens", "refs", "free_pages", "n_free", "scratch")]
    + [{"scratch": A[5] + 4}, {"refs": A[0] + 4 * 31}, {"free_pages": A[2] + 196}, {"n_free": A[3] + 4}, {"scratch": A[1]}])
def test_page_pool_refusals(built_lib, change):
    refused(-8, "b2_page_pool", b2.page_pool, **{**POOL, **change})


COMPACT = dict(table=A[0], table_stride=8, lens=A[1], n_req=4, page_size=16, max_pages=8, refs=A[2], n_pages=50,
               pairs=A[3], max_pairs=25, info=A[4], scratch=A[5])


@pytest.mark.parametrize("change", [
    {"n_req": 0}, {"n_req": 16385}, {"page_size": 0}, {"n_pages": 0}, {"max_pages": 0}, {"max_pairs": 0}, {"table_stride": 7}]
    + [{k: 0} for k in ("table", "lens", "refs", "pairs", "info", "scratch")]
    + [{k: P + 2} for k in ("table", "lens", "refs", "pairs", "info", "scratch")]
    + [{"pairs": A[2] + 196}, {"table": A[1]}, {"info": A[3] + 296}, {"scratch": A[2]}])
def test_page_compact_refusals(built_lib, change):
    refused(-8, "b2_page_compact", b2.page_compact, **{**COMPACT, **change})


def test_rows_beside_rows_are_apart(built_lib):
    """The old and the new table as the halves of each row of one buffer: told
    apart, so the refusal that follows is that of the device."""
    with pytest.raises(b2.B2Error) as e:
        b2.page_fork(**{**FORK, "table_stride": 16, "new_stride": 16, "new_table": A[1] + 32})
    assert "overlaps" not in str(e.value)
    refused(-8, "overlaps", b2.page_fork, **{**FORK, "table_stride": 16, "new_stride": 16, "new_table": A[1] + 28})
    refused(-8, "overlaps", b2.page_fork, **{**FORK, "table_stride": 15, "new_stride": 16, "new_table": A[1] + 32})


OPTS = dict(dtype=b2.F16, nh=4, n_req=4, max_pages=8)


@pytest.mark.parametrize("change,code", [
    ({"dtype": b2.BF16}, -3), ({"dtype": 2}, -3), ({"nh": 3}, -8), ({"nh": 0}, -8), ({"n_req": 3}, -8), ({"n_req": 0}, -8),
    ({"max_pages": 0}, -8), ({"len_add": -1}, -8), ({"window": -1}, -8), ({"scale": -1.0}, -8),
    ({"scale": math.nan}, -8), ({"softcap": math.inf}, -8), ({"out_stride": 255}, -8), ({"q_stride": -8}, -8),
    ({"table_stride": 7}, -8)])
def test_attention_shared_refusals(built_lib, change, code):
    o = b2.paged_attn_opts(**{**OPTS, **change})
    refused(code, "b2_attention_shared", b2.attention_shared, kv(), o, P, P, P, 0, 4, P, P, 2, P, 0, P)


def test_attention_shared_null_refusals(built_lib):
    o = b2.paged_attn_opts(**OPTS)
    for i in (2, 3, 4, 6, 7, 8, 9, 10, 12):
        a = [kv(), o, P, P, P, 0, 4, P, P, 2, P, 0, P]
        a[i] = 0
        refused(-8, "b2_attention_shared", b2.attention_shared, *a)
    for i in (2, 3, 4, 5, 7, 8, 10, 11, 12):
        a = [kv(), o, P, P, P, P, 4, P, P, 2, P, P, P]
        a[i] = P + 1
        refused(-8, "aligned", b2.attention_shared, *a)
    refused(-8, "b2_attention_shared", b2.attention_shared, kv(hd=60), o, P, P, P, 0, 4, P, P, 2, P, 0, P)
