"""b2_attention_shared without a GPU: what it writes may not share memory with what
it reads, and is told apart from what only lies beside it."""
import pytest

import b2decode as b2

# addresses that no refused call reads, far enough apart for every size below
A = [(i + 1) << 32 for i in range(16)]
ROWS, NH, NKV, HD, PAGES, P, MAX = 6, 8, 2, 64, 10, 16, 5
IN = {"q": 2 * NH * HD * ROWS, "table": 4 * MAX * 4, "lens": 4 * ROWS, "req": 4 * ROWS, "starts": 4 * 4, "prefix": 4 * 3,
      "slopes": 4 * NH, "k": 2 * PAGES * P * NKV * HD, "v": 2 * PAGES * P * NKV * HD}
OUT = {"out": 2 * NH * HD * ROWS, "lse": 4 * NH * ROWS, "scratch": 4096}
AT = dict(zip([*IN, *OUT], A))


def call(strides=None, cache=None, **at):
    a = {**AT, **at}
    kv = b2.paged_kv(a["k"], a["v"], b2.F16, PAGES, P, NKV, HD, *(cache or ()))
    o = b2.paged_attn_opts(b2.F16, NH, 4, MAX, slopes=a["slopes"], **(strides or {}))
    with pytest.raises(b2.B2Error) as e:
        b2.attention_shared(kv, o, a["q"], a["table"], a["lens"], a["req"], ROWS, a["starts"], a["prefix"], 3, a["out"], a["lse"],
                            a["scratch"])
    return e.value.code, str(e.value)


@pytest.mark.parametrize("out", OUT)
@pytest.mark.parametrize("name", IN)
def test_outputs_that_meet_inputs(built_lib, out, name):
    for at in (AT[name], AT[name] + IN[name] - 16 if IN[name] % 16 == 0 else AT[name], AT[name] - OUT[out] + 16):
        code, text = call(**{out: at})
        assert code == -8 and "b2_attention_shared" in text and f"{out} overlaps" in text, text
    end = AT[name] + (IN[name] + 15) // 16 * 16
    for at in (end, AT[name] - OUT[out]) if out != "scratch" else (end,):
        assert "overlaps" not in call(**{out: at})[1]


def test_outputs_that_meet_outputs(built_lib):
    for a, b in (("out", "lse"), ("lse", "scratch"), ("scratch", "out")):
        code, text = call(**{a: AT[b]})
        assert code == -8 and "overlaps" in text
    assert "overlaps" not in call(lse=AT["out"] + OUT["out"])[1]
    assert "overlaps" not in call()[1]


def test_rows_beside_rows_are_apart(built_lib):
    """q and out as parts of each row of one buffer; out between the pages of a cache with room between them."""
    row = NH * HD
    s = dict(q_stride=3 * row, out_stride=3 * row)
    assert "overlaps" not in call(s, out=AT["q"] + 2 * row)[1]
    assert "out overlaps q" in call(s, out=AT["q"] + 2 * row - 16)[1]
    wide = (1 << 20, NKV * HD, HD)
    assert "overlaps" not in call(cache=wide, out=AT["k"] + 2 * P * NKV * HD)[1]
    assert "out overlaps the cache's k" in call(cache=wide, out=AT["k"] + (2 << 20) * 3 - 16)[1]


def test_inputs_may_be_one_another(built_lib):
    assert "overlaps" not in call(prefix=AT["lens"], starts=AT["lens"], q=AT["k"], v=AT["k"])[1]
