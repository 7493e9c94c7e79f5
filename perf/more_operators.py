"""The operators of a beam search over a paged cache: cases, inputs, plain forms, work and 64-bit values.

A step of a server that keeps several continuations of each request, its KV cache in pages, runs, in this order:

  beam_select       the best continuations over a request's beams and the vocabulary, the token histories reordered
  page_fork         block tables of the beams that go on, the pages that they must not share copied, the free list
  attention_shared  attention of rows that share a prefix (beams, a common system prompt, a prompt's own tokens)
  page_compact      now and then: the pages in use moved to the front of the pool

`run` computes them with elementary torch operations where `own` is false, and
through the framework's entry points where it is true.
"""
import math
import os
import sys

import numpy as np
import torch

own = False

F32, F16, BF16 = 0, 1, 30  # ggml type ids, as the framework names types
_TORCH = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_ID = {"f32": F32, "f16": F16, "bf16": BF16}
_SIZE = {"f32": 4, "f16": 2, "bf16": 2}
_ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------

def _beam(name, groups, width, n, pad, dtype, k, eos, history, dead=0.0, masked=0.0):
    return {"name": name, "op": "beam_select", "groups": groups, "width": width, "n": n, "pad": pad, "dtype": dtype,
            "k": k, "eos": eos, "history": history, "dead": dead, "masked": masked}


def _fork(name, groups, width, prompt_min, prompt_max, new, page, layers, nkv, hd, cache):
    return {"name": name, "op": "page_fork", "groups": groups, "width": width, "prompt_min": prompt_min,
            "prompt_max": prompt_max, "new": new, "page": page, "layers": layers, "nkv": nkv, "hd": hd, "cache": cache}


def _compact(name, pages, used, rows, page, layers, nkv, hd, cache):
    return {"name": name, "op": "page_compact", "pages": pages, "used": used, "rows": rows, "page": page,
            "layers": layers, "nkv": nkv, "hd": hd, "cache": cache}


def _attn(name, groups, rows_min, rows_max, prefix_min, prefix_max, suffix_min, suffix_max, causal, nh, nkv, hd, dtype,
          cache, page, softcap=0.0, window=0, alibi=False):
    return {"name": name, "op": "attention_shared", "groups": groups, "rows_min": rows_min, "rows_max": rows_max,
            "prefix_min": prefix_min, "prefix_max": prefix_max, "suffix_min": suffix_min, "suffix_max": suffix_max,
            "causal": causal, "nh": nh, "nkv": nkv, "hd": hd, "dtype": dtype, "cache": cache, "page": page,
            "softcap": softcap, "window": window, "alibi": alibi}


def listed():
    return [
        # one request with 4 beams over Qwen2.5's vocabulary, histories of up to 4096 tokens: latency counts
        _beam("beam-1x4-152k", 1, 4, 151936, 0, "f32", 4, 151643, 4096),
        # the framework's largest batch as two requests of 8 beams, Llama-3's vocabulary, some beams ended, rows padded
        _beam("beam-2x8-128k-masked", 2, 8, 128256, 64, "f32", 8, 128009, 8192, dead=0.2, masked=0.1),
        # a server's 64 requests of 16 beams, 16-bit logits, twice as many candidates as beams
        _beam("beam-64x16-128k", 64, 16, 128256, 0, "bf16", 32, 128009, 1024),
        # 4 beams of one request, all 24 layers of the 0.5B shape
        _fork("fork-1x4-05b", 1, 4, 2000, 2000, 37, 16, 24, 2, 64, "f16"),
        # 16 requests of 8 beams, all 32 layers of the 8B shape
        _fork("fork-16x8-8b", 16, 8, 40, 700, 21, 16, 32, 8, 128, "f16"),
        # a small pool's leftovers, the 0.5B shape
        _compact("compact-512-05b", 512, 0.5, 16, 16, 24, 2, 64, "f16"),
        # a long-running server's pool, half empty, four layers of the 8B shape
        _compact("compact-8192-8b", 8192, 0.55, 96, 16, 4, 8, 128, "bf16"),
        # beams of one request of the 8B heads, fp32 rows over the fp16 cache as the engine keeps them: latency counts
        _attn("shared-1x4-2k-f32", 1, 4, 4, 2000, 2000, 33, 33, False, 32, 8, 128, "f32", "f16", 16),
        # 16 requests of 1 to 8 beams of the 0.5B heads, ragged prompts, a cap on the scores and a sliding window
        _attn("shared-16-ragged-cap", 16, 1, 8, 24, 9001, 0, 300, False, 14, 2, 64, "bf16", "bf16", 24, softcap=30.0,
              window=4096),
        # 8 requests of 8 beams of the 8B heads, prompts of 1K to 32K, fp32 rows
        _attn("shared-8x8-32k-f32", 8, 8, 8, 1024, 32768, 16, 512, False, 32, 8, 128, "f32", "f16", 16),
        # 64 conversations of the 72B heads behind one system prompt of 32K
        _attn("shared-1x64-32k-72b", 1, 64, 64, 32768, 32768, 16, 2048, False, 64, 8, 128, "bf16", "bf16", 16),
        # a prompt of 2048 tokens of the 72B heads: its rows share the prompt's own positions
        _attn("shared-prompt-2k-72b", 1, 2048, 2048, 2048, 2048, 0, 0, True, 64, 8, 128, "bf16", "bf16", 16),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["beam_select", "page_fork", "page_compact", "attention_shared", "attention_shared"])
    cache = rng.choice(["f16", "bf16"])
    page = rng.choice([1, 8, 16, 24, 32, 64, 100])
    if op == "beam_select":
        n = _log_int(rng, 100, 152064)
        dtype = rng.choice(["f32", "f16", "bf16"])
        width = _log_int(rng, 1, 32)
        most = 1024 * 128256 * 2 // (n * (4 if dtype == "f32" else 2))
        groups = _log_int(rng, 1, max(1, min(256, most // width)))
        case = _beam("", groups, width, n, rng.choice([0, 0, 1, 8, 64, 77]), dtype,
                     min(64, n // 2, rng.choice([width, width, 2 * width])), rng.choice([-1, rng.randrange(n)]),
                     _log_int(rng, 1, 8192), rng.choice([0.0, 0.0, 0.3]), rng.choice([0.0, 0.0, 0.1, 0.5]))
    elif op == "page_fork":
        layers, nkv, hd = rng.choice([(24, 2, 64), (32, 8, 128), (8, 8, 128), (1, 1, 80), (3, 4, 96), (80, 1, 128)])
        groups, width = _log_int(rng, 1, 64), _log_int(rng, 1, 16)
        page = max(8, page)
        hi = _log_int(rng, 1, 8192)
        case = _fork("", groups, width, _log_int(rng, 1, hi), hi, _log_int(rng, 1, 200), page, layers, nkv, hd, cache)
        while _fork_pages(case) * page * nkv * hd * 4 * layers > 2 << 30:  # what the case's pool takes
            case["prompt_max"] = max(1, case["prompt_max"] // 2)
            case["prompt_min"] = min(case["prompt_min"], case["prompt_max"])
            case["groups"] = max(1, case["groups"] // 2)
            case["new"] = max(1, case["new"] // 2)
    elif op == "page_compact":
        layers, nkv, hd = rng.choice([(24, 2, 64), (32, 8, 128), (8, 8, 128), (1, 1, 80), (3, 4, 96), (80, 1, 128)])
        pages = _log_int(rng, 4, 65536)
        while pages * page * nkv * hd * 4 * layers > 2 << 30:
            pages //= 2
        case = _compact("", max(2, pages), rng.uniform(0.02, 0.98), _log_int(rng, 1, 512), page, layers, nkv, hd, cache)
    else:
        hd = rng.choice([32, 64, 64, 80, 96, 128, 128])
        nkv = rng.choice([1, 2, 4, 8])
        nh = nkv * rng.choice([1, 2, 4, 7, 8, 16])
        dtype = rng.choice(["f32", "f16", "bf16"])
        if dtype != "f32":
            cache = dtype
        causal = rng.random() < 0.3
        groups, rows = _log_int(rng, 1, 64), _log_int(rng, 1, 2048 if causal else 128)
        prefix = _log_int(rng, 1, 32768)
        suffix = rng.choice([0, _log_int(rng, 1, 2048)])
        while True:  # no dearer than the largest listed case
            total = groups * rows
            if total * nh * (prefix + suffix) <= 64 * 64 * 33792 and groups * (prefix + rows * suffix) * nkv * hd <= 1 << 27:
                break
            groups, rows = max(1, groups // 2), max(1, rows * 3 // 4)
            prefix, suffix = max(1, prefix * 3 // 4), suffix * 3 // 4
        case = _attn("", groups, _log_int(rng, 1, rows), rows, _log_int(rng, 1, prefix), prefix,
                     0 if causal else rng.randint(0, suffix), 0 if causal else suffix, causal, nh, nkv, hd, dtype, cache,
                     page, rng.choice([0.0, 0.0, 30.0, 50.0]), rng.choice([0, 0, _log_int(rng, 1, 8192)]),
                     rng.random() < 0.25)
    del case["name"]
    return case


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------

def _spread(lo, hi, n):
    """n whole numbers from lo to hi, even over the logarithm."""
    if n == 1:
        return [hi]
    return [int(round((lo + 1) * ((hi + 1) / (lo + 1)) ** (i / (n - 1)))) - 1 for i in range(n)]


def _prepare_beam(case, seed, dev):
    g = torch.Generator(device=dev).manual_seed(seed)
    G, W, n, k = case["groups"], case["width"], case["n"], case["k"]
    rows, ld, dt = G * W, n + case["pad"], _TORCH[case["dtype"]]
    x = torch.empty(rows, ld, device=dev, dtype=dt)
    x.normal_(0.0, 2.5, generator=g)
    # a model is sure of a few tokens
    peaks = (torch.randint(0, n, (rows, 1), device=dev, generator=g) + torch.arange(4, device=dev) * (n // 5 + 1)) % n
    x.scatter_add_(1, peaks, (6.0 * torch.rand(rows, 4, device=dev, generator=g) + 4.0).to(dt))
    if case["masked"]:
        x[:, :n].masked_fill_(torch.rand(rows, n, device=dev, generator=g) < case["masked"], -math.inf)
    scores = -4.0 * torch.rand(rows, device=dev, generator=g) - 10.0 * torch.rand(G, 1, device=dev, generator=g).expand(
        G, W).reshape(rows)
    if case["dead"]:  # beams that have ended; a request keeps one at least
        dead = (torch.rand(G, W, device=dev, generator=g) < case["dead"]) & (torch.arange(W, device=dev) > 0)
        scores.masked_fill_(dead.reshape(rows), -math.inf)
    H = case["history"]
    lens = torch.randint(0, H, (G, 1), device=dev, generator=g).expand(G, W).reshape(rows).to(torch.int32)
    new = lambda t, *s: torch.zeros(*s, device=dev, dtype=t)  # noqa: E731
    return {"x": x, "scores": scores, "hist": torch.randint(0, n, (rows, H), device=dev, generator=g, dtype=torch.int32),
            "lens": lens, "parent": new(torch.int32, G, k), "token": new(torch.int32, G, k),
            "score": new(torch.float32, G, k), "eos_score": new(torch.float32, rows),
            "new_hist": new(torch.int32, G * k, H), "new_lens": new(torch.int32, G * k)}


def _fork_pages(case):
    """Pages that the beams of a fork case hold, at most, and a few more."""
    P = case["page"]
    held = sum(n // P + case["width"] * (case["new"] // P + 3) for n in _spread(case["prompt_min"], case["prompt_max"],
                                                                             case["groups"]))
    return held + case["groups"] * case["width"] + 4


def _parents(case, r):
    """The beam that each beam continues: a few carry most of the continuations, now and then one finds none."""
    G, W = case["groups"], case["width"]
    weight = r.random((G, W)) ** 3
    parent = np.stack([np.sort(r.choice(W, W, p=w / w.sum())) + g * W for g, w in enumerate(weight)]).reshape(-1)
    return np.where(r.random(G * W) < 0.02, -1, parent) if W > 2 else parent


def _prepare_fork(case, seed, dev):
    r = np.random.default_rng(seed)
    G, W, P = case["groups"], case["width"], case["page"]
    prompts = _spread(case["prompt_min"], case["prompt_max"], G)
    n_pages = _fork_pages(case)
    ids = r.permutation(n_pages).astype(np.int32)
    max_pages = (max(prompts) + case["new"]) // P + 2
    table = np.full((G * W, max_pages), -1, np.int32)
    lens = np.zeros(G * W, np.int32)
    at = 0
    for g in range(G):  # the prompt's full pages are shared, the rest is each beam's own
        n = prompts[g] + int(r.integers(1, case["new"] + 1))
        full, all_ = prompts[g] // P, -(-n // P)
        for w in range(W):
            table[g * W + w, :full] = ids[at:at + full]
        at += full
        for w in range(W):
            table[g * W + w, full:all_] = ids[at:at + all_ - full]
            at += all_ - full
        lens[g * W:(g + 1) * W] = n
    parent = _parents(case, r)
    refs = np.bincount(table[table >= 0], minlength=n_pages)
    free = np.flatnonzero(refs == 0)
    up = lambda a: torch.from_numpy(np.ascontiguousarray(a)).to(dev, torch.int32)  # noqa: E731
    none = lambda *s: torch.full(s, -1, device=dev, dtype=torch.int32)  # noqa: E731
    cache = torch.empty(case["layers"], 2, n_pages, P, case["nkv"], case["hd"], device=dev, dtype=_TORCH[case["cache"]])
    cache.normal_(generator=torch.Generator(device=dev).manual_seed(seed))
    free_list = none(n_pages)
    free_list[:len(free)] = up(free)
    return {"parent": up(parent), "table": up(table), "lens": up(lens), "refs": up(refs), "free": free_list,
            "n_free": up(np.array([len(free)])), "cache": cache, "new_table": none(*table.shape),
            "new_lens": none(G * W), "pairs": none(G * W, 3), "info": none(4), "new_refs": none(n_pages),
            "new_free": none(n_pages), "new_n_free": none(1)}


def _held(N, used, r):
    """The pages in use, in the order in which the requests hold them; recent requests hold the high ones."""
    held = np.argsort(r.random(N) ** (1.0 + np.arange(N) / N))[:used].astype(np.int32)
    r.shuffle(held)
    return held


def _used(case):
    return min(case["pages"], max(1, int(round(case["used"] * case["pages"]))))


def _prepare_compact(case, seed, dev):
    r = np.random.default_rng(seed)
    N, P, R = case["pages"], case["page"], case["rows"]
    used = _used(case)
    held = _held(N, used, r)
    weight = 16.0 ** (np.arange(R) / R)  # short requests and long ones
    ends = np.floor(np.cumsum(weight) / weight.sum() * used + 1e-9).astype(np.int64)
    ends[-1] = used
    sizes = np.diff(np.concatenate([[0], ends]))
    most = int(sizes.max())
    cuts = np.concatenate([[0], np.cumsum(r.permutation(sizes))])
    shared = min(2, most)
    table = np.full((R, most + shared), -1, np.int32)
    lens = np.zeros(R, np.int32)
    head = held[:shared]
    for i in range(R):
        mine = held[cuts[i]:cuts[i + 1]]
        row = np.concatenate([head, mine]) if i % 3 == 1 and len(mine) else mine  # some begin with a common prefix
        table[i, :len(row)] = row
        lens[i] = max(0, len(row) * P - (int(r.integers(0, P)) if len(row) else 0))
    refs = np.bincount(table[table >= 0], minlength=N)
    up = lambda a: torch.from_numpy(np.ascontiguousarray(a)).to(dev, torch.int32)  # noqa: E731
    cache = torch.empty(case["layers"], 2, N, P, case["nkv"], case["hd"], device=dev, dtype=_TORCH[case["cache"]])
    cache.normal_(generator=torch.Generator(device=dev).manual_seed(seed))
    return {"table": up(table), "lens": up(lens), "refs": up(refs), "cache": cache,
            "pairs": torch.full((max(1, N // 2), 3), -1, device=dev, dtype=torch.int32),
            "info": torch.zeros(4, device=dev, dtype=torch.int32)}


def _attn_shape(case):
    """Per group: rows, shared positions, and the positions that each row sees beside them (behind them)."""
    rows = _spread(case["rows_min"], case["rows_max"], case["groups"])
    prefix = _spread(case["prefix_min"], case["prefix_max"], case["groups"])
    rows = [max(1, n) for n in rows]
    prefix = [max(n, p, 1) if case["causal"] else p // case["page"] * case["page"] for n, p in zip(rows, prefix)]
    lens = []
    for n, p in zip(rows, prefix):
        if case["causal"]:  # the last n positions of a sequence of p
            lens.append([p - n + 1 + i for i in range(n)])
        else:
            lens.append([p + s for s in _spread(case["suffix_min"], case["suffix_max"], n)])
    return rows, prefix, lens


def _prepare_attn(case, seed, dev):
    g = torch.Generator(device=dev).manual_seed(seed)
    r = np.random.default_rng(seed)
    nh, nkv, hd, P = case["nh"], case["nkv"], case["hd"], case["page"]
    rows, prefix, lens = _attn_shape(case)
    B = sum(rows)
    tables, at, most = [], 0, max(-(-max(n) // P) for n in lens) + 1
    for n, p, ls in zip(rows, prefix, lens):
        full = -(-p // P)
        shared = np.arange(at, at + full)
        at += full
        for ln in ls[:1] if case["causal"] else ls:
            own_pages = max(0, -(-ln // P) - full)
            tables.append(np.concatenate([shared, np.arange(at, at + own_pages), np.full(most - full - own_pages, -1)]))
            at += own_pages
    pool = at + 3
    ids = np.append(r.permutation(pool), -1)
    table = torch.from_numpy(ids[np.stack(tables).astype(np.int64)]).to(dev, torch.int32)
    req = np.repeat(np.arange(len(rows)), rows) if case["causal"] else np.arange(B)
    cache = torch.empty(2, pool, P, nkv, hd, device=dev, dtype=_TORCH[case["cache"]])
    cache.normal_(generator=g)
    dt = _TORCH[case["dtype"]]
    up = lambda a: torch.tensor(a, device=dev, dtype=torch.int32)  # noqa: E731
    s = {"q": (1.5 * torch.randn(B, nh, hd, device=dev, generator=g)).to(dt), "cache": cache, "table": table,
         "req": up(req), "lens": up([x for ls in lens for x in ls]), "starts": up(np.cumsum([0] + rows)),
         "prefix": up(prefix), "shape": (rows, prefix, lens), "out": torch.empty(B, nh, hd, device=dev, dtype=dt),
         "lse": torch.empty(B, nh, device=dev)}
    if case["alibi"]:
        s["slopes"] = 2.0 ** (-8.0 * torch.arange(1, nh + 1, device=dev, dtype=torch.float32) / nh)
    return s


_PREPARE = {"beam_select": _prepare_beam, "page_fork": _prepare_fork, "page_compact": _prepare_compact,
            "attention_shared": _prepare_attn}


def prepare(case, seed):
    s = _PREPARE[case["op"]](case, int(seed), torch.device("cuda"))
    s["case"] = dict(case)
    return s


# ---------------------------------------------------------------------------
# the plain forms
# ---------------------------------------------------------------------------

def _plain_beam(s):
    c = s["case"]
    G, W, n, k = c["groups"], c["width"], c["n"], c["k"]
    x = s["x"][:, :n].double()  # the order of close candidates needs 64 bits
    m = x.amax(-1, keepdim=True)
    d = x - m
    lp = s["scores"].double()[:, None] + (d - torch.log(torch.exp(d).sum(-1, keepdim=True)))
    if c["eos"] >= 0:
        s["eos_score"].copy_(lp[:, c["eos"]])
        lp[:, c["eos"]] = -math.inf
    val, at = torch.sort(lp.view(G, W * n), dim=1, descending=True, stable=True)
    val, at = val[:, :k], at[:, :k]
    ok = val > -math.inf
    row = torch.arange(G, device=x.device)[:, None] * W + at // n
    s["parent"].copy_(torch.where(ok, row, -1))
    s["token"].copy_(torch.where(ok, at % n, -1))
    s["score"].copy_(val)
    H = c["history"]
    par, tok = s["parent"].view(-1).long(), s["token"].view(-1)
    live, src = par >= 0, par.clamp(min=0)
    ln = s["lens"][src].long()
    col = torch.arange(H, device=x.device)[None, :]
    new = torch.where(col < ln[:, None], s["hist"][src], torch.where(col == ln[:, None], tok[:, None], s["new_hist"]))
    s["new_hist"].copy_(torch.where(live[:, None], new, s["new_hist"]))
    s["new_lens"].copy_(torch.where(live, (ln + 1).clamp(max=H), 0))
    return _beam_out(s)


def _beam_out(s):
    return {n: s[n] for n in ("parent", "token", "score", "eos_score", "new_hist", "new_lens")}


def _plain_pool(table, lens, page, n_pages):
    """How many rows hold each page, and the pages that none holds."""
    col = torch.arange(table.shape[1], device=table.device)[None, :]
    held = table[(col < (lens.long()[:, None] + page - 1) // page) & (table >= 0)].long()
    refs = torch.zeros(n_pages, device=table.device, dtype=torch.int32).index_add_(
        0, held, torch.ones_like(held, dtype=torch.int32))
    return refs, torch.nonzero(refs == 0)[:, 0]


def _plain_fork(s):
    P, par = s["case"]["page"], s["parent"].long()
    dev = par.device
    R, n_pages = par.numel(), s["refs"].numel()
    live, src = par >= 0, par.clamp(min=0)
    lens = torch.where(live, s["lens"][src].long(), 0)
    old = s["table"][src]
    col = torch.arange(old.shape[1], device=dev)[None, :]
    s["new_table"].copy_(torch.where(col < ((lens + P - 1) // P)[:, None], old, s["new_table"]))
    part = lens % P != 0
    last = old[torch.arange(R, device=dev), (lens // P).clamp(max=old.shape[1] - 1)].long()
    same = (par[:, None] == par[None, :]) & live[None, :]
    first = ~(same & (torch.arange(R, device=dev)[None, :] < torch.arange(R, device=dev)[:, None])).any(1)
    copies = live & part & ~(first & (s["refs"][last.clamp(min=0)] <= 1))
    who = torch.nonzero(copies)[:, 0]
    n = who.numel()
    page = s["free"][:n]
    s["new_table"][who, lens[who] // P] = page
    s["pairs"][:n] = torch.stack([last[who], page.long(), lens[who] % P], 1).to(torch.int32)
    s["new_lens"].copy_(lens)
    s["info"].copy_(torch.tensor([0, n, 0, 0], device=dev))
    _plain_copy(s["cache"], s["pairs"][:n])
    refs, free = _plain_pool(s["new_table"], s["new_lens"], P, n_pages)
    s["new_refs"].copy_(refs)
    s["new_free"][:free.numel()] = free.to(torch.int32)
    s["new_n_free"].fill_(free.numel())
    return _fork_out(s)


def _plain_copy(cache, pairs):
    src, dst, n = pairs.long().unbind(1)
    if src.numel() == 0:
        return
    keep = torch.arange(cache.shape[3], device=cache.device)[None, :] < n[:, None]
    for layer in cache:
        for kv in layer:
            kv[dst] = torch.where(keep[:, :, None, None], kv[src], kv[dst])


def _fork_out(s):
    return {n: s[n] for n in ("new_table", "new_lens", "pairs", "info", "cache", "new_refs", "new_free", "new_n_free")}


def _plain_compact(s):
    P, refs, table = s["case"]["page"], s["refs"], s["table"]
    used = torch.nonzero(refs > 0)[:, 0]
    U = used.numel()
    movers = used[used >= U].flip(0)
    holes = torch.nonzero(refs[:U] == 0)[:, 0]
    n = movers.numel()
    to = torch.arange(refs.numel(), device=refs.device)
    to[movers] = holes
    col = torch.arange(table.shape[1], device=table.device)[None, :]
    held = (col < (s["lens"].long()[:, None] + P - 1) // P) & (table >= 0)
    table.copy_(torch.where(held, to[table.clamp(min=0).long()].to(torch.int32), table))
    s["pairs"][:n] = torch.stack([movers, holes, torch.full_like(holes, P)], 1).to(torch.int32)
    s["info"].copy_(torch.tensor([0, n, U, U], device=table.device))
    _plain_copy(s["cache"], s["pairs"][:n])
    return _compact_out(s)


def _compact_out(s):
    return {n: s[n] for n in ("table", "pairs", "info", "cache")}


def _plain_attn(s):
    c = s["case"]
    nh, nkv, hd, P = c["nh"], c["nkv"], c["hd"], c["page"]
    dev = s["q"].device
    kc, vc = s["cache"].view(2, -1, nkv, hd)

    def places(rows, lo, hi):  # of positions [lo, hi) in the tables' rows
        j = torch.arange(lo, hi, device=dev)
        return rows[:, j // P].long().clamp(min=0) * P + j % P

    at = 0
    for n, p, lens in zip(*s["shape"]):
        q = s["q"][at:at + n].float().view(n, nkv, nh // nkv, hd)
        tab = s["table"][s["req"][at:at + n].long()]
        ln = s["lens"][at:at + n].long()
        most = max(lens)
        if most == 0:  # nothing cached yet
            s["out"][at:at + n].zero_()
            s["lse"][at:at + n].fill_(-math.inf)
            at += n
            continue
        slot = places(tab[:1], 0, p)[0]
        sc = [torch.einsum("rkgd,jkd->rkgj", q, kc[slot].float())]
        if most > p:
            own_slot = places(tab, p, most)
            sc.append(torch.matmul(q, kc[own_slot].float().permute(0, 2, 3, 1)))
        sc = torch.cat(sc, 3) * hd ** -0.5
        j = torch.arange(sc.shape[3], device=dev)
        if c["softcap"]:
            sc = c["softcap"] * torch.tanh(sc / c["softcap"])
        if c["alibi"]:
            sc = sc + s["slopes"].view(1, nkv, -1, 1) * (j[None, :] - (ln[:, None] - 1)).float()[:, None, None, :]
        seen = j[None, :] < ln[:, None]
        if c["window"]:
            seen = seen & (j[None, :] >= ln[:, None] - c["window"])
        sc = sc.masked_fill(~seen[:, None, None, :], -math.inf)
        m = sc.amax(-1, keepdim=True)
        e = torch.exp(sc - torch.where(m > -math.inf, m, 0.0))
        z = e.sum(-1, keepdim=True)
        o = torch.einsum("rkgj,jkd->rkgd", e[..., :p], vc[slot].float())
        if most > p:
            o = o + torch.matmul(e[..., p:], vc[own_slot].float().permute(0, 2, 1, 3))
        s["out"][at:at + n].copy_(torch.where(z > 0, o / z, 0.0).reshape(n, nh, hd))
        s["lse"][at:at + n].copy_((m + torch.log(z)).reshape(n, nh))
        at += n
    return {"out": s["out"], "lse": s["lse"]}


_PLAIN = {"beam_select": _plain_beam, "page_fork": _plain_fork, "page_compact": _plain_compact,
          "attention_shared": _plain_attn}


# ---------------------------------------------------------------------------
# the framework's entry points
# ---------------------------------------------------------------------------

def _lib():
    path = os.path.join(_ROOT, "ai-agent-framework_b200")
    if path not in sys.path:
        sys.path.insert(0, path)
    import b2decode
    return b2decode


def _stream():
    return torch.cuda.current_stream().cuda_stream


def _scratch(s, nbytes):
    if "scratch" not in s:
        s["scratch"] = torch.empty(max(16, nbytes()), device="cuda", dtype=torch.uint8)
    return s["scratch"].data_ptr()


def _kv(s, b2, cache):
    """The cache's description (its first layer), made once as a server makes it."""
    if "kv" not in s:
        k, v = cache
        s["kv"] = b2.paged_kv(k.data_ptr(), v.data_ptr(), _ID[s["case"]["cache"]], *k.shape)
    return s["kv"]


def _own_beam(s, b2):
    c, x = s["case"], s["x"]
    G, W, k, H = c["groups"], c["width"], c["k"], c["history"]
    scratch = _scratch(s, lambda: b2.beam_select_scratch_bytes(c["n"], G, W, k))
    b2.beam_select(x.data_ptr(), _ID[c["dtype"]], c["n"], G, W, x.stride(0), s["scores"].data_ptr(), k, c["eos"],
                   s["parent"].data_ptr(), s["token"].data_ptr(), s["score"].data_ptr(),
                   s["eos_score"].data_ptr() if c["eos"] >= 0 else 0, scratch, _stream())
    b2.beam_reorder(s["hist"].data_ptr(), G * W, H, s["new_hist"].data_ptr(), G * k, H, H, s["parent"].data_ptr(),
                    s["lens"].data_ptr(), s["token"].data_ptr(), s["new_lens"].data_ptr(), _stream())
    return _beam_out(s)


def _own_fork(s, b2):
    c, t, cache = s["case"], s["table"], s["cache"]
    R, N = s["parent"].numel(), s["refs"].numel()
    scratch = _scratch(s, lambda: b2.page_pool_scratch_bytes(N))
    b2.page_fork(s["parent"].data_ptr(), R, t.data_ptr(), t.stride(0), s["lens"].data_ptr(), t.shape[0], c["page"],
                 s["refs"].data_ptr(), N, s["free"].data_ptr(), s["n_free"].data_ptr(), s["new_table"].data_ptr(),
                 s["new_table"].stride(0), t.shape[1], s["new_lens"].data_ptr(), s["pairs"].data_ptr(),
                 s["info"].data_ptr(), _stream())
    b2.page_copy(_kv(s, b2, cache[0]), c["layers"], cache.stride(0), s["pairs"].data_ptr(), s["info"].data_ptr() + 4, R,
                 _stream())
    b2.page_pool(s["new_table"].data_ptr(), s["new_table"].stride(0), s["new_lens"].data_ptr(), R, c["page"], t.shape[1],
                 s["new_refs"].data_ptr(), N, s["new_free"].data_ptr(), s["new_n_free"].data_ptr(), scratch, _stream())
    return _fork_out(s)


def _own_compact(s, b2):
    c, t, cache = s["case"], s["table"], s["cache"]
    N = s["refs"].numel()
    scratch = _scratch(s, lambda: b2.page_compact_scratch_bytes(N))
    b2.page_compact(t.data_ptr(), t.stride(0), s["lens"].data_ptr(), t.shape[0], c["page"], t.shape[1],
                    s["refs"].data_ptr(), N, s["pairs"].data_ptr(), s["pairs"].shape[0], s["info"].data_ptr(), scratch,
                    _stream())
    b2.page_copy(_kv(s, b2, cache[0]), c["layers"], cache.stride(0), s["pairs"].data_ptr(), s["info"].data_ptr() + 4,
                 s["pairs"].shape[0], _stream())
    return _compact_out(s)


def _own_attn(s, b2):
    c = s["case"]
    B, t = s["q"].shape[0], s["table"]
    if "opts" not in s:
        s["opts"] = b2.paged_attn_opts(_ID[c["dtype"]], c["nh"], t.shape[0], t.shape[1], softcap=c["softcap"],
                                       window=c["window"], slopes=s["slopes"].data_ptr() if c["alibi"] else 0)
    scratch = _scratch(s, lambda: b2.attention_shared_scratch_bytes(B, c["nh"], c["nkv"], c["hd"]))
    b2.attention_shared(_kv(s, b2, s["cache"]), s["opts"], s["q"].data_ptr(), t.data_ptr(), s["lens"].data_ptr(),
                        s["req"].data_ptr(), B, s["starts"].data_ptr(), s["prefix"].data_ptr(), c["groups"],
                        s["out"].data_ptr(), s["lse"].data_ptr(), scratch, _stream())
    return {"out": s["out"], "lse": s["lse"]}


_OWN = {"beam_select": _own_beam, "page_fork": _own_fork, "page_compact": _own_compact, "attention_shared": _own_attn}


def run(state):
    op = state["case"]["op"]
    if own:
        return _OWN[op](state, _lib())
    return _PLAIN[op](state)


# ---------------------------------------------------------------------------
# work of one pass: each input read once, each output written once
# ---------------------------------------------------------------------------

def work(case):
    op = case["op"]
    if op == "beam_select":
        rows = case["groups"] * case["width"]
        out = case["groups"] * case["k"]
        # (histories of half their room on average, read and written)
        return {"bytes": rows * (case["n"] * _SIZE[case["dtype"]] + 12) + out * (12 + 4 + 4 * case["history"]),
                "flops": 4 * rows * case["n"]}
    if op == "page_fork":
        P, W = case["page"], case["width"]
        rows = case["groups"] * W
        entries = sum(W * (-(-(n + case["new"] // 2) // P)) for n in _spread(case["prompt_min"], case["prompt_max"],
                                                                            case["groups"]))
        # beams that do not continue alone, half a page each on average
        parent = _parents(case, np.random.default_rng(0))
        copies = (parent >= 0).sum() - len(np.unique(parent[parent >= 0]))
        moved = copies * (P / 2) * case["nkv"] * case["hd"] * 4 * case["layers"]
        return {"bytes": int(2 * moved + 8 * entries + 12 * rows + 12 * _fork_pages(case)), "flops": 0}
    if op == "page_compact":
        N, u = case["pages"], _used(case)
        moves = int((_held(N, u, np.random.default_rng(0)) >= u).sum())
        moved = moves * case["page"] * case["nkv"] * case["hd"] * 4 * case["layers"]
        return {"bytes": int(2 * moved + 4 * N + 8 * u + 12 * moves), "flops": 0}
    nh, nkv, hd = case["nh"], case["nkv"], case["hd"]
    rows, prefix, lens = _attn_shape(case)
    read = seen = 0
    for p, ls in zip(prefix, lens):
        first = [max(0, n - case["window"]) if case["window"] else 0 for n in ls]
        read += max(0, max(min(n, p) for n in ls) - min(first))
        read += sum(max(0, n - max(p, f)) for n, f in zip(ls, first))
        seen += sum(n - f for n, f in zip(ls, first))
    B = sum(rows)
    return {"bytes": 2 * read * nkv * hd * 2 + 2 * B * nh * hd * _SIZE[case["dtype"]] + 4 * B * nh
            + 4 * (read // case["page"] + 2 * B), "flops": 4 * seen * nh * hd}


# ---------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------

def _exact_beam(case, s):
    G, W, n, k, H = case["groups"], case["width"], case["n"], case["k"], case["history"]
    out = {"parent": [], "token": [], "score": []}
    eos = s["eos_score"].double()
    new_hist, new_lens = s["new_hist"].clone(), s["new_lens"].clone()
    for g in range(G):
        best = []
        for r in range(g * W, (g + 1) * W):
            if s["scores"][r] == -math.inf:
                if case["eos"] >= 0:
                    eos[r] = -math.inf
                continue
            lp = torch.log_softmax(s["x"][r, :n].double(), 0) + s["scores"][r].double()
            if case["eos"] >= 0:
                eos[r] = lp[case["eos"]]
                lp[case["eos"]] = -math.inf
            v, i = torch.sort(lp, descending=True, stable=True)
            best += [(-a, r, b) for a, b in zip(v[:k].tolist(), i[:k].tolist()) if a > -math.inf]
        best = sorted(best)[:k]
        best += [(math.inf, -1, -1)] * (k - len(best))
        for e, (v, r, t) in enumerate(best):
            if r >= 0:
                ln = int(s["lens"][r])
                row = torch.cat([s["hist"][r, :ln], torch.tensor([t], device=s["x"].device, dtype=torch.int32)])[:H]
                new_hist[g * k + e, :len(row)] = row
                new_lens[g * k + e] = len(row)
            else:
                new_lens[g * k + e] = 0
        for name, at, sign in (("score", 0, -1), ("parent", 1, 1), ("token", 2, 1)):
            out[name].append([sign * b[at] for b in best])
    dev = s["x"].device
    return {"parent": torch.tensor(out["parent"], device=dev, dtype=torch.int32),
            "token": torch.tensor(out["token"], device=dev, dtype=torch.int32),
            "score": torch.tensor(out["score"], device=dev, dtype=torch.float64), "eos_score": eos,
            "new_hist": new_hist, "new_lens": new_lens}


def _exact_attn(case, s):
    nh, nkv, hd, P = case["nh"], case["nkv"], case["hd"], case["page"]
    out, lse = [], []
    for b, (r, n) in enumerate(zip(s["req"].tolist(), s["lens"].tolist())):
        first = max(0, n - case["window"]) if case["window"] else 0
        if n == 0:
            out.append(torch.zeros(nh, hd, device=s["q"].device, dtype=torch.float64))
            lse.append(torch.full((nh,), -math.inf, device=s["q"].device, dtype=torch.float64))
            continue
        pages = s["table"][r, first // P:(n + P - 1) // P].long()
        k, v = (c[pages].reshape(-1, nkv, hd)[first % P:first % P + n - first].double() for c in s["cache"])
        q = s["q"][b].double().view(nkv, nh // nkv, hd)
        sc = torch.matmul(q, k.permute(1, 2, 0)).view(nh, -1) / math.sqrt(hd)
        if case["softcap"]:
            sc = torch.tanh(sc / case["softcap"]) * case["softcap"]
        if case["alibi"]:
            sc = sc - s["slopes"].double()[:, None] * torch.arange(n - first - 1, -1, -1, device=sc.device)
        z = torch.logsumexp(sc, 1)
        w = torch.exp(sc - z[:, None]).view(nkv, nh // nkv, -1)
        out.append(torch.matmul(w, v.permute(1, 0, 2)).view(nh, hd))
        lse.append(z)
    return {"out": torch.stack(out), "lse": torch.stack(lse)}


def exact(case, seed):
    if case["op"] == "beam_select":
        return _exact_beam(case, prepare(case, seed))
    if case["op"] == "attention_shared":
        return _exact_attn(case, prepare(case, seed))
    return None  # whole numbers and copies: the plain form says what they are
