"""The documented step of a beam search, taken from the text that a user reads and
run against whole-number models of the page operators: after every step each
row writes a page of its own."""
import glob
import os
import types

import numpy as np
import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
START = "A step of a beam search over the same cache"


def documented_step():
    text = next(t for t in (open(p).read() for p in sorted(glob.glob(os.path.join(ROOT, "*.md")))) if START in t)
    return text[text.index(START):].split("```python\n")[1].split("```")[0]


class Mem:
    """Device words: an address that whole words can be added to."""

    def __init__(self, a):
        self.a = a

    def __add__(self, nbytes):
        return Mem(self.a.reshape(-1)[nbytes // 4:])


def ints(*shape):
    return Mem(np.zeros(shape, np.int32))


def page_pool(table, stride, lens, n_req, P, max_pages, refs, n_pages, free, n_free, scratch, stream):
    held = np.concatenate([table.a[r, :-(-int(lens.a[r]) // P)] for r in range(n_req)])
    refs.a[:] = np.bincount(held, minlength=n_pages)
    f = np.flatnonzero(refs.a == 0)
    free.a[:len(f)] = f
    n_free.a[0] = len(f)


def page_fork(parent, n_req, table, stride, lens, n_src, P, refs, n_pages, free, n_free, new_table, new_stride, max_pages,
              new_lens, pairs, info, stream):
    seen, taken = set(), 0
    for r in range(n_req):
        p = int(parent.a[r])
        n = int(lens.a[p])
        new_lens.a[r] = n
        new_table.a[r, :-(-n // P)] = table.a[p, :-(-n // P)]
        if n % P and (p in seen or refs.a[table.a[p, n // P]] > 1):
            page = free.a[taken]
            pairs.a[taken] = table.a[p, n // P], page, n % P
            new_table.a[r, n // P] = page
            taken += 1
        seen.add(p)
    assert taken <= n_free.a[0]
    info.a[:] = 0, taken, 0, 0


def page_plan(cached, fresh, n_req, P, free, n_free, table, stride, max_pages, lens, starts, slots, positions, token_req,
              max_tokens, info, stream):
    taken = 0
    for r in range(n_req):
        n = int(cached.a[r])
        if n % P == 0:
            table.a[r, n // P] = free.a[taken]
            taken += 1
        lens.a[r] = n + 1
        slots.a[r] = table.a[r, n // P] * P + n % P
    assert taken <= n_free.a[0] and (fresh.a == 1).all()
    info.a[:] = 0, n_req, taken, 0


@pytest.mark.parametrize("P,G,W,first", [(4, 1, 2, 4), (4, 2, 3, 6), (16, 3, 4, 31), (1, 2, 2, 1)])
def test_documented_step_gives_each_row_a_page_to_write(P, G, W, first):
    g = np.random.default_rng(P)
    R, max_pages = G * W, first // P + 30
    n_pages = R * max_pages
    written = {}  # slot -> what the last token there continues

    def page_copy(kv, layers, stride, pairs, n_pairs, max_pairs, stream):
        for s, d, n in pairs.a[:n_pairs.a[0]].tolist():
            assert s != d
            for i in range(n):
                written[d * P + i] = written[s * P + i]

    def beam_select(*a):
        parent.a[:] = np.concatenate([np.sort(g.integers(0, W, W)) + W * i for i in range(G)])

    def copy(dst, src, nbytes, stream):
        dst.a.reshape(-1)[:nbytes // 4] = src.a.reshape(-1)[:nbytes // 4]

    ignore = lambda *a: None  # noqa: E731
    b2decode = types.SimpleNamespace(F32=0, page_fork=page_fork, page_copy=page_copy, page_pool=page_pool, page_plan=page_plan,
                                     attention_shared=ignore, beam_select=beam_select, beam_reorder=ignore)
    parent, table, lens, refs, free, n_free = ints(R), ints(R, max_pages), ints(R), ints(n_pages), ints(n_pages), ints(1)
    ns = {"b2decode": b2decode, "copy": copy, "parent": parent, "R": R, "G": G, "W": W, "table": table, "max_pages": max_pages,
          "lens": lens, "page_size": P, "refs": refs, "n_pages": n_pages, "free_pages": free, "n_free": n_free,
          "new_table": ints(R, max_pages), "new_lens": ints(R), "pairs": ints(R, 3), "info": ints(4), "cached": ints(R),
          "fresh": Mem(np.ones(R, np.int32)), "starts": ints(R + 1), "slots": ints(R), "positions": ints(R), "token_req": ints(R),
          "plan_info": ints(4), "layers": 1, "vocab": 9, "room": 64}
    for name in ("kv_layer0", "layer_stride", "stream", "scratch", "kv", "opts", "q_rot", "groups", "prefix", "out", "logits", "scores",
                 "eos", "token", "score", "eos_score", "history", "new_history", "history_lens", "new_history_lens"):
        ns[name] = 0
    # the beams of a request share the pages of `first` positions, the last one in part
    tails = [[("prompt", i // W, j) for j in range(first)] for i in range(R)]
    for r in range(R):
        pages = np.arange(-(-first // P)) + r // W * max_pages
        table.a[r, :len(pages)] = pages
        lens.a[r] = first
        for j in range(first):
            written[int(pages[j // P]) * P + j % P] = tails[r][j]
    page_pool(table, max_pages, lens, R, P, max_pages, refs, n_pages, free, n_free, 0, 0)
    beam_select()
    step = compile(documented_step(), "the documented step", "exec")
    for t in range(20):
        chosen = parent.a.copy()
        ns["cached"].a[:] = -99
        exec(step, ns)
        assert ns["info"].a[0] == 0 and ns["plan_info"].a[0] == 0
        slots = ns["slots"].a.tolist()
        assert len({s // P for s in slots}) == R, (t, slots)
        tails = [tails[chosen[r]] + [(t, r)] for r in range(R)]
        now = ns["table"]  # what the next step continues
        for r in range(R):
            written[slots[r]] = (t, r)
        for r in range(R):
            n = int(ns["lens"].a[r])
            assert [written[int(now.a[r, j // P]) * P + j % P] for j in range(n)] == tails[r], (t, r)
