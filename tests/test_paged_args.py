"""The paged serving operators without a GPU: every refusal of their entry
points comes before the first CUDA call, so it is the same with and without a
device; b2_rope_freqs is host arithmetic and is compared with its formulas."""
import math

import numpy as np
import pytest

import b2decode as b2
from conftest import has_gpu

P = 4096  # an address that no refused call reads


def refused(code, text, fn, *args, **kw):
    with pytest.raises(b2.B2Error) as e:
        fn(*args, **kw)
    assert e.value.code == code and text in str(e.value), str(e.value)


def kv(**kw):
    a = dict(k_ptr=P, v_ptr=P, dtype=b2.F16, n_pages=4, page_size=16, nkv=2, hd=64)
    a.update(kw)
    return b2.paged_kv(**a)


PLAN = dict(cached=P, fresh=P, n_req=4, page_size=16, free_pages=P, n_free=P, table=P, table_stride=8, max_pages=8,
            lens=P, starts=P, slots=P, positions=P, token_req=P, max_tokens=4, info=P)


@pytest.mark.parametrize("change", [
    {"n_req": 0}, {"n_req": -1}, {"n_req": 16385}, {"page_size": 0}, {"max_pages": 0}, {"max_tokens": 0},
    {"table_stride": 7}] + [{k: None} for k in ("cached", "fresh", "free_pages", "n_free", "table", "lens", "starts",
                                                "slots", "positions", "token_req", "info")])
def test_page_plan_refusals(built_lib, change):
    refused(-8, "b2_page_plan", b2.page_plan, **{**PLAN, **change})


ROWS = dict(dtype=b2.F16, nh=4, nkv=2, hd=64, rot_dim=64)


@pytest.mark.parametrize("change,code", [
    ({"dtype": 8}, -3), ({"hd": 63}, -8), ({"hd": 0}, -8), ({"hd": 258}, -8), ({"nh": -1}, -8), ({"nh": 0}, -8),
    ({"rot_dim": 63}, -8), ({"rot_dim": 66}, -8), ({"rot_dim": -2}, -8), ({"layout": 2}, -8), ({"q_stride": -1}, -8),
    ({"q_out_stride": 255}, -8), ({"k_out_stride": 127}, -8)])
def test_rope_row_refusals(built_lib, change, code):
    rows = b2.rope_rows(**{**ROWS, **change})
    refused(code, "b2_rope", b2.rope, rows, P, P, 3, q=P, k=P, q_out=P, k_out=P)
    refused(code, "b2_rope_append", b2.rope_append, rows, kv(), P, P, P, 3, P, P, P, P)


@pytest.mark.parametrize("args", [
    dict(freqs=0), dict(positions=0), dict(n_tok=0), dict(q_out=0), dict(k=0), dict(k_out=0), dict(q=0)])
def test_rope_null_refusals(built_lib, args):
    a = dict(freqs=P, positions=P, n_tok=3, q=P, k=P, q_out=P, k_out=P)
    refused(-8, "b2_rope", b2.rope, b2.rope_rows(**ROWS), **{**a, **args})
    refused(-8, "b2_rope", b2.rope, b2.rope_rows(**ROWS), P, P, 3)


@pytest.mark.parametrize("change,code", [
    ({"k_ptr": 0}, -8), ({"v_ptr": 0}, -8), ({"dtype": b2.F32}, -3), ({"n_pages": 0}, -8), ({"page_size": 0}, -8),
    ({"nkv": 0}, -8), ({"hd": 60}, -8), ({"hd": 264}, -8), ({"k_ptr": P + 8}, -8),
    ({"page_stride": 2048, "pos_stride": 130, "head_stride": 64}, -8),
    ({"page_stride": -2048, "pos_stride": 128, "head_stride": 64}, -8)])
def test_paged_cache_refusals(built_lib, change, code):
    o = b2.paged_attn_opts(b2.F16, 4, 4, 8)
    refused(code, "b2_attention_paged", b2.attention_paged, kv(**change), o, P, P, P, 0, 4, P, 0, P)
    refused(code, "b2_rope_append", b2.rope_append, b2.rope_rows(**ROWS), kv(**change), P, P, P, 3, P, P, P, P)


def test_rope_append_refusals(built_lib):
    rows = b2.rope_rows(**ROWS)
    for change in ({"nkv": 4}, {"hd": 128}):
        refused(-8, "do not match", b2.rope_append, rows, kv(**change), P, P, P, 3, P, P, P, P)
    refused(-3, "cache's type", b2.rope_append, rows, kv(dtype=b2.BF16), P, P, P, 3, P, P, P, P)
    for i in range(3, 8):  # positions, slots, n_tok, q_out without q, ...
        a = [rows, kv(), P, P, P, 3, P, P, P, P]
        a[i] = 0
        refused(-8, "b2_rope_append", b2.rope_append, *a)


OPTS = dict(dtype=b2.F16, nh=4, n_req=4, max_pages=8)


@pytest.mark.parametrize("change,code", [
    ({"dtype": b2.BF16}, -3), ({"dtype": 2}, -3), ({"nh": 3}, -8), ({"nh": 0}, -8), ({"n_req": 3}, -8), ({"n_req": 0}, -8),
    ({"max_pages": 0}, -8), ({"len_add": -1}, -8), ({"window": -1}, -8), ({"scale": -1.0}, -8),
    ({"scale": math.nan}, -8), ({"scale": math.inf}, -8), ({"softcap": -1.0}, -8), ({"softcap": math.nan}, -8),
    ({"out_stride": 255}, -8), ({"q_stride": -8}, -8), ({"table_stride": 7}, -8)])
def test_attention_paged_refusals(built_lib, change, code):
    o = b2.paged_attn_opts(**{**OPTS, **change})
    refused(code, "b2_attention_paged", b2.attention_paged, kv(), o, P, P, P, 0, 4, P, 0, P)


def test_attention_paged_null_refusals(built_lib):
    for i in (2, 3, 4, 6, 7, 9):
        a = [kv(), b2.paged_attn_opts(**OPTS), P, P, P, 0, 4, P, 0, P]
        a[i] = 0
        refused(-8, "b2_attention_paged", b2.attention_paged, *a)
    refused(-8, "aligned", b2.attention_paged, kv(), b2.paged_attn_opts(**OPTS), P, P, P, 0, 4, P, 0, P + 4)
    for a in ((0, 4, 2, 64), (4, 3, 2, 64), (4, 4, 0, 64), (4, 4, 2, 512)):
        refused(-8, "scratch", b2.attention_paged_scratch_bytes, *a)


ODD = P + 1


def test_misaligned_pointers(built_lib):
    """Addresses that the element types do not allow, told before any of them is used."""
    for name in ("cached", "fresh", "free_pages", "n_free", "table", "lens", "starts", "slots", "positions", "token_req", "info"):
        refused(-8, "aligned", b2.page_plan, **{**PLAN, name: ODD})
    refused(-8, "aligned", b2.page_plan, **{**PLAN, "slots": P + 4})
    for name in ("freqs", "positions", "q", "k", "q_out", "k_out"):
        a = dict(freqs=P, positions=P, n_tok=3, q=P, k=P, q_out=P, k_out=P)
        refused(-8, "aligned", b2.rope, b2.rope_rows(**ROWS), **{**a, name: ODD})
    refused(-8, "aligned", b2.rope, b2.rope_rows(**{**ROWS, "dtype": b2.F32}), P, P, 3, q=P + 2, q_out=P)
    for i in (2, 3, 4, 6, 7, 8, 9):
        a = [b2.rope_rows(**ROWS), kv(), P, P, P, 3, P, P, P, P]
        a[i] = ODD
        refused(-8, "aligned", b2.rope_append, *a)
    for i in (2, 3, 4, 5, 7, 8, 9):
        a = [kv(), b2.paged_attn_opts(**OPTS), P, P, P, P, 4, P, P, P]
        a[i] = ODD
        refused(-8, "aligned", b2.attention_paged, *a)
    refused(-8, "aligned", b2.attention_paged, kv(), b2.paged_attn_opts(**OPTS, slopes=ODD), P, P, P, 0, 4, P, 0, P)
    for name in ("logits", "ids", "logprob", "entropy", "top_ids", "top_logprob"):
        refused(-8, "aligned", b2.logprobs, **{**LOGP, name: ODD})


LOGP = dict(logits=P, dtype=b2.F32, n=100, rows=2, ld=100, ids=P, m=1, logprob=P, entropy=P, k=5, top_ids=P, top_logprob=P)


@pytest.mark.parametrize("change,code", [
    ({"logits": None}, -8), ({"dtype": 8}, -3), ({"n": 0}, -8), ({"n": (1 << 30) + 1, "ld": 1 << 31}, -8), ({"rows": 0}, -8),
    ({"ld": 99}, -8), ({"m": -1}, -8), ({"k": -1}, -8), ({"k": 65}, -8), ({"k": 20, "n": 10}, -8), ({"ids": 0}, -8),
    ({"logprob": 0}, -8), ({"top_ids": 0}, -8), ({"top_logprob": 0}, -8)])
def test_logprobs_refusals(built_lib, change, code):
    refused(code, "b2_logprobs", b2.logprobs, **{**LOGP, **change})


def test_batch_logprobs_without_a_batch(built_lib):
    assert built_lib.b2_batch_logprobs(None, 1, None, 0, None, None, 0, None, None) == -10


@pytest.mark.skipif(has_gpu(), reason="checks the no-GPU error path")
def test_no_gpu_is_an_error(built_lib):
    refused(-5, "no CUDA device", b2.page_plan, **PLAN)
    refused(-5, "no CUDA device", b2.rope, b2.rope_rows(**ROWS), P, P, 3, q=P, k=P, q_out=P, k_out=P)
    refused(-5, "no CUDA device", b2.attention_paged, kv(), b2.paged_attn_opts(**OPTS), P, P, P, 0, 4, P, 0, P)
    refused(-5, "no CUDA device", b2.logprobs, **LOGP)
    refused(-5, "no CUDA device", b2.attention_paged_scratch_bytes, 4, 4, 2, 64)


def _freqs(rot, theta, scaling, f, ctx, low, high):
    i = np.arange(rot // 2, dtype=np.float64)
    base = theta ** (-2 * i / rot)
    if scaling == b2.ROPE_SCALE_NONE:
        return base
    if scaling == b2.ROPE_SCALE_LINEAR:
        return base / f
    if scaling == b2.ROPE_SCALE_BANDS:
        keep = (ctx * base / (2 * np.pi) - low) / (high - low)
    else:
        def pair(t):
            return rot * np.log(ctx / (t * 2 * np.pi)) / (2 * np.log(theta))
        a, b = max(np.floor(pair(high)), 0), min(np.ceil(pair(low)), rot - 1)
        keep = 1 - (i - a) / max(b - a, 1e-3)
    keep = np.clip(keep, 0, 1)
    return base * (keep + (1 - keep) / f)


@pytest.mark.parametrize("rot", [2, 6, 64, 128, 256])
@pytest.mark.parametrize("scaling", [0, 1, 2, 3])
def test_rope_freqs(built_lib, rot, scaling):
    for theta, f, ctx in ((10000.0, 4.0, 4096.0), (500000.0, 8.0, 8192.0), (1e6, 1.5, 32768.0)):
        for low, high in ((0.0, 0.0), (2.0, 16.0)):
            got, scale = b2.rope_freqs(rot, theta, scaling, f, ctx, low, high)
            want = _freqs(rot, theta, scaling, f, ctx, low or 1.0, high or (32.0 if scaling == 3 else 4.0))
            # one pow (half a step or so each side) and four roundings
            np.testing.assert_allclose(got, want, rtol=8 * np.finfo(np.float64).eps)
            assert scale == (np.float32(0.1 * math.log(f) + 1) if scaling == 3 else 1.0)


@pytest.mark.parametrize("kw", [
    dict(rot_dim=0, theta=1e4), dict(rot_dim=7, theta=1e4), dict(rot_dim=64, theta=1.0), dict(rot_dim=64, theta=math.nan),
    dict(rot_dim=64, theta=1e4, scaling=4), dict(rot_dim=64, theta=1e4, scaling=1, factor=0.0),
    dict(rot_dim=64, theta=1e4, scaling=2, factor=2.0), dict(rot_dim=64, theta=1e4, scaling=3, factor=2.0, orig_ctx=-1.0),
    dict(rot_dim=64, theta=1e4, scaling=2, factor=2.0, orig_ctx=4096, low=4.0, high=4.0)])
def test_rope_freqs_refusals(built_lib, kw):
    refused(-8, "b2_rope_freqs", b2.rope_freqs, **kw)
