"""The operators of a paged serving step: their cases, inputs, plain forms, work and 64-bit values.

A step of a server that keeps its KV cache in pages runs, in this order:

  plan             block tables and slot maps of the step's tokens, from request lengths
  rope_append      rotary positions on q and k, k and v written into their cache slots
  attention_paged  attention of one query row per sequence over the paged cache
  logprobs         log probabilities of given tokens, entropy and the top alternatives

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
_ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------

def _plan(name, n_req, tokens, max_cached, page):
    return {"name": name, "op": "plan", "n_req": n_req, "tokens": tokens, "max_cached": max_cached, "page": page}


def _rope(name, tokens, nh, nkv, hd, rot, layout, dtype, cache, scaling, theta, factor, context, page):
    return {"name": name, "op": "rope_append", "tokens": tokens, "nh": nh, "nkv": nkv, "hd": hd, "rot": rot,
            "layout": layout, "dtype": dtype, "cache": cache, "scaling": scaling, "theta": theta, "factor": factor,
            "context": context, "page": page}


def _attn(name, batch, nh, nkv, hd, ctx_min, ctx_max, dtype, cache, page, softcap=0.0, window=0, alibi=False):
    return {"name": name, "op": "attention_paged", "batch": batch, "nh": nh, "nkv": nkv, "hd": hd, "ctx_min": ctx_min,
            "ctx_max": ctx_max, "dtype": dtype, "cache": cache, "page": page, "softcap": softcap, "window": window,
            "alibi": alibi}


def _logp(name, rows, n, pad, dtype, m, k, masked):
    return {"name": name, "op": "logprobs", "rows": rows, "n": n, "pad": pad, "dtype": dtype, "m": m, "k": k,
            "masked": masked}


def listed():
    return [
        # a decode step of the framework's largest batch: 16 sequences, one new token each
        _plan("plan-16x1", 16, 16, 8192, 16),
        # a step that admits prompts beside running sequences: many requests, a million tokens
        _plan("plan-2048-1M", 2048, 1048576, 32768, 16),
        # one decode step's rows of Llama-3-8B (interleaved pairs, as the engine rotates), fp32 rows, fp16 cache
        _rope("rope-16-8b-f32", 16, 32, 8, 128, 128, "interleaved", "f32", "f16", "none", 500000.0, 1.0, 8192, 16),
        # a mixed step of Qwen2.5-0.5B heads: half layout, half of the head rotated, positions stretched 4 times
        _rope("rope-517-05b-half", 517, 14, 2, 64, 32, "half", "bf16", "bf16", "linear", 1000000.0, 4.0, 131072, 24),
        # a long prompt of the 72B heads, positions scaled per wavelength for a context of 128K
        _rope("rope-32k-72b-yarn", 32768, 64, 8, 128, 128, "half", "bf16", "bf16", "yarn", 1000000.0, 4.0, 131072, 16),
        # the decode attention's own shapes: one sequence of 4K, where latency counts, ...
        _attn("attn-1x4k-f32", 1, 32, 8, 128, 4096, 4096, "f32", "f16", 16),
        # ... Qwen2.5-0.5B heads, ragged lengths from one token on, a cap on the scores and a sliding window
        _attn("attn-16-ragged-cap", 16, 14, 2, 64, 1, 9001, "bf16", "bf16", 24, softcap=30.0, window=4096),
        # ... 64 sequences of the 72B heads from 16 tokens to 16K (a server's usual mix)
        _attn("attn-64-ragged-72b", 64, 64, 8, 128, 16, 16384, "bf16", "bf16", 16),
        # ... and eight sequences of 32K, the largest of the attention benchmark
        _attn("attn-8x32k-f32", 8, 32, 8, 128, 32768, 32768, "f32", "f16", 64),
        # the token just sampled of one sequence, with 20 alternatives, over Qwen2.5's vocabulary
        _logp("logp-1x152k", 1, 151936, 0, "f32", 1, 20, 0.0),
        # a batched step's 16 rows, a tenth of the vocabulary masked out, rows padded, 4 candidates each
        _logp("logp-16x128k-masked", 16, 128256, 64, "f32", 4, 5, 0.1),
        # scores of a prompt: 2048 positions, one given token each and the best alternative
        _logp("logp-2048x128k", 2048, 128256, 0, "bf16", 1, 1, 0.0),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["plan", "rope_append", "attention_paged", "logprobs"])
    if op == "plan":
        n_req = _log_int(rng, 1, 4096)
        tokens = _log_int(rng, 1, 1048576)
        case = _plan("", n_req, tokens, _log_int(rng, 1, 32768), rng.choice([1, 8, 16, 24, 32, 64, 100, 128, 256]))
        while case["tokens"] // case["page"] > 65536:  # no more pages than the largest listed case takes
            case["tokens"] //= 2
        while n_req * (case["max_cached"] // case["page"]) > 2048 * 2048:  # and no larger a table
            case["max_cached"] //= 2
    elif op == "rope_append":
        hd = rng.choice([32, 64, 80, 96, 128, 192, 256])
        nkv = rng.choice([1, 2, 4, 8])
        nh = nkv * rng.choice([1, 2, 4, 7, 8])
        rot = rng.choice([hd, hd // 2, hd // 4, 2 * rng.randint(1, hd // 2)])
        rot -= rot % 2
        dtype = rng.choice(["f32", "f16", "bf16"])
        cache = dtype if dtype != "f32" else rng.choice(["f16", "bf16"])
        most = 32768 * 80 * 128 * 2 // ((nh + 2 * nkv) * hd * (4 if dtype == "f32" else 2))
        scaling = rng.choice(["none", "linear", "bands", "yarn"])
        case = _rope("", _log_int(rng, 1, max(1, min(32768, most))), nh, nkv, hd, max(2, rot),
                     rng.choice(["interleaved", "half"]), dtype, cache, scaling,
                     rng.choice([10000.0, 500000.0, 1000000.0]), 1.0 if scaling == "none" else rng.choice([2.0, 4.0, 8.0]),
                     rng.choice([4096, 32768, 131072, 1000000]), rng.choice([1, 8, 16, 24, 64, 100]))
    elif op == "attention_paged":
        hd = rng.choice([32, 64, 80, 96, 128, 192, 256])
        nkv = rng.choice([1, 2, 4, 8])
        nh = nkv * rng.choice([1, 2, 4, 7, 8, 16, 20])
        dtype = rng.choice(["f32", "f16", "bf16"])
        cache = dtype if dtype != "f32" else rng.choice(["f16", "bf16"])
        batch = _log_int(rng, 1, 256)
        ctx_max = _log_int(rng, 1, 65536)
        while batch * ctx_max * nkv * hd > 8 * 32768 * 8 * 128 or batch * ctx_max * nh > 8 * 32768 * 32:
            ctx_max = max(1, ctx_max // 2)
            if ctx_max < 4096:
                batch = max(1, batch // 2)
        case = _attn("", batch, nh, nkv, hd, _log_int(rng, 1, ctx_max), ctx_max, dtype, cache,
                     rng.choice([1, 8, 16, 24, 64, 100]), rng.choice([0.0, 0.0, 30.0, 50.0]),
                     rng.choice([0, 0, _log_int(rng, 1, 8192)]), rng.random() < 0.25)
    else:
        n = _log_int(rng, 100, 152064)
        dtype = rng.choice(["f32", "f16", "bf16"])
        most = 2048 * 128256 * 2 // (n * (4 if dtype == "f32" else 2))
        case = _logp("", _log_int(rng, 1, min(4096, most)), n, rng.choice([0, 0, 1, 8, 64, 77]), dtype,
                     rng.choice([0, 1, 1, 2, 8]), rng.choice([0, 1, 5, 20, 32]), rng.choice([0.0, 0.0, 0.1, 0.9]))
    del case["name"]
    return case


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------

def _lens(case):
    """The sequences' lengths of an attention case: spread evenly over the logarithm."""
    b, lo, hi = case["batch"], case["ctx_min"], case["ctx_max"]
    return [hi if b == 1 else int(round(lo * (hi / lo) ** (i / (b - 1)))) for i in range(b)]


def _freqs(case):
    """Radians per position of each pair, and the factor on cos and sin."""
    rot, theta, f = case["rot"], case["theta"], case["factor"]
    i = np.arange(rot // 2, dtype=np.float64)
    base = theta ** (-2.0 * i / rot)
    if case["scaling"] == "none":
        return base, 1.0
    if case["scaling"] == "linear":
        return base / f, 1.0
    original = case["context"] / f
    if case["scaling"] == "bands":  # long wavelengths stretched, short ones kept, a linear blend between
        turns = original * base / (2 * math.pi)
        keep = np.clip((turns - 1.0) / (4.0 - 1.0), 0.0, 1.0)
        return base * (keep + (1.0 - keep) / f), 1.0
    # yarn: the blend is linear in the pair's number, between the pairs that turn 32 times and once
    def pair(turns):
        return rot * math.log(original / (turns * 2 * math.pi)) / (2 * math.log(theta))
    lo, hi = max(math.floor(pair(32.0)), 0), min(math.ceil(pair(1.0)), rot - 1)
    keep = 1.0 - np.clip((i - lo) / max(hi - lo, 1e-3), 0.0, 1.0)
    return base * (keep + (1.0 - keep) / f), 0.1 * math.log(f) + 1.0


def _most_fresh(case):
    return min(case["tokens"], 8 * (case["tokens"] // case["n_req"] + 1))


def _prepare_plan(case, seed, dev):
    g = np.random.default_rng(seed)
    R, T, P = case["n_req"], case["tokens"], case["page"]
    cached = np.exp(g.uniform(0.0, math.log(case["max_cached"] + 1.0), R)).astype(np.int64) - 1
    cached = np.clip(cached, 0, case["max_cached"])
    if T == R:  # a decode step
        fresh = np.ones(R, dtype=np.int64)
    else:  # some requests idle, the others share the step's tokens unevenly
        share = np.minimum(np.exp(g.normal(0.0, 1.0, R)), 6.0) * (g.random(R) < 0.9)
        share[g.integers(R)] += 1.0
        share = np.minimum(share / share.mean(), 7.0)
        ends = np.floor(np.cumsum(share) / share.sum() * T + 1e-9).astype(np.int64)
        ends[-1] = T
        fresh = np.minimum(np.diff(np.concatenate([[0], ends])), _most_fresh(case))
        while fresh.sum() < T:  # what the cap took goes to the requests below it
            below = np.flatnonzero(fresh < _most_fresh(case))
            more = min(T - int(fresh.sum()), len(below))
            fresh[below[:more]] += 1
    have, total = -(-cached // P), -(-(cached + fresh) // P)
    need = int((total - have).sum())
    max_pages = (case["max_cached"] + _most_fresh(case)) // P + 3
    ids = g.permutation(int(total.sum()) + 64).astype(np.int32)
    held, free = ids[:int(have.sum())], ids[int(have.sum()):]
    table = np.full((R, max_pages), -1, dtype=np.int32)
    table[np.arange(max_pages)[None, :] < have[:, None]] = held
    up = lambda a, t: torch.from_numpy(np.ascontiguousarray(a)).to(dev, t)  # noqa: E731
    new = lambda n, t: torch.empty(n, device=dev, dtype=t)  # noqa: E731
    cap = T + 5  # the step's token rows, the last of them padding
    assert need <= len(free)
    return {"cached": up(cached, torch.int32), "fresh": up(fresh, torch.int32), "free": up(free, torch.int32),
            "n_free": up([len(free)], torch.int32), "table": up(table, torch.int32), "cap": cap,
            "lens": new(R, torch.int32), "starts": new(R + 1, torch.int32), "slots": new(cap, torch.int64),
            "positions": new(cap, torch.int32), "token_req": new(cap, torch.int32), "info": new(4, torch.int32)}


def _prepare_rope(case, seed, dev):
    g = torch.Generator(device=dev).manual_seed(seed)
    T, nh, nkv, hd, P = case["tokens"], case["nh"], case["nkv"], case["hd"], case["page"]
    dt, ct = _TORCH[case["dtype"]], _TORCH[case["cache"]]
    qkv = torch.randn(T, (nh + 2 * nkv) * hd, device=dev, generator=g).to(dt)  # one projection's rows
    pages = -(-T // P) + 8
    cache = torch.zeros(2, pages, P, nkv, hd, device=dev, dtype=ct)
    slots = torch.randperm(pages * P, device=dev, generator=g)[:T]
    if T > 8:
        slots[-(T // 64 + 1):] = -1  # padding rows of a step of fixed size
    run = max(1, T // 8)  # runs of consecutive positions, each from somewhere in the context
    first = torch.randint(0, max(1, case["context"] - run), (8,), device=dev, generator=g)
    t = torch.arange(T, device=dev)
    positions = (first[(t // run) % 8] + t % run).to(torch.int32)
    freqs, scale = _freqs(case)
    return {"q": qkv[:, :nh * hd].view(T, nh, hd), "k": qkv[:, nh * hd:(nh + nkv) * hd].view(T, nkv, hd),
            "v": qkv[:, (nh + nkv) * hd:].view(T, nkv, hd), "positions": positions, "slots": slots, "cache": cache,
            "freqs": torch.from_numpy(freqs).to(dev), "scale": scale,
            "q_out": torch.empty(T, nh, hd, device=dev, dtype=dt)}


def _prepare_attn(case, seed, dev):
    g = torch.Generator(device=dev).manual_seed(seed)
    B, nh, nkv, hd, P = case["batch"], case["nh"], case["nkv"], case["hd"], case["page"]
    lens = torch.tensor(_lens(case))[torch.randperm(B, generator=torch.Generator().manual_seed(seed))]
    n_pages = (lens + P - 1) // P
    max_pages = int(n_pages.max()) + 1
    total = int(n_pages.sum())
    pool = total + 4
    cache = torch.empty(2, pool, P, nkv, hd, device=dev, dtype=_TORCH[case["cache"]])
    cache.normal_(generator=g)
    ids = torch.randperm(pool, device=dev, generator=g)[:total].to(torch.int32)
    table = torch.full((B, max_pages), -1, device=dev, dtype=torch.int32)
    table[torch.arange(max_pages, device=dev)[None, :] < n_pages.to(dev)[:, None]] = ids
    dt = _TORCH[case["dtype"]]
    s = {"q": (1.5 * torch.randn(B, nh, hd, device=dev, generator=g)).to(dt), "cache": cache, "table": table,
         "lens": lens.to(dev, torch.int32), "max_len": int(lens.max()),
         "out": torch.empty(B, nh, hd, device=dev, dtype=dt), "lse": torch.empty(B, nh, device=dev)}
    if case["alibi"]:
        s["slopes"] = 2.0 ** (-8.0 * torch.arange(1, nh + 1, device=dev, dtype=torch.float32) / nh)
    return s


def _prepare_logp(case, seed, dev):
    g = torch.Generator(device=dev).manual_seed(seed)
    rows, n, ld = case["rows"], case["n"], case["n"] + case["pad"]
    dt = _TORCH[case["dtype"]]
    x = torch.empty(rows, ld, device=dev, dtype=dt)
    x.normal_(0.0, 2.5, generator=g)
    # a model is sure of a few tokens
    peaks = (torch.randint(0, n, (rows, 1), device=dev, generator=g) + torch.arange(4, device=dev) * (n // 5 + 1)) % n
    x.scatter_add_(1, peaks, (6.0 * torch.rand(rows, 4, device=dev, generator=g) + 4.0).to(dt))
    if case["masked"]:
        x[:, :n].masked_fill_(torch.rand(rows, n, device=dev, generator=g) < case["masked"], -math.inf)
    m, k = case["m"], case["k"]
    ids = torch.randint(0, n, (rows, m), device=dev, generator=g)
    if m:
        ids[:, 0] = torch.where(torch.rand(rows, device=dev, generator=g) < 0.7, peaks[:, 0], ids[:, 0])
    new = lambda *s: torch.empty(*s, device=dev)  # noqa: E731
    return {"x": x, "ids": ids.to(torch.int32), "logprob": new(rows, m), "entropy": new(rows),
            "top_ids": torch.empty(rows, k, device=dev, dtype=torch.int32), "top_logprob": new(rows, k)}


_PREPARE = {"plan": _prepare_plan, "rope_append": _prepare_rope, "attention_paged": _prepare_attn,
            "logprobs": _prepare_logp}


def prepare(case, seed):
    s = _PREPARE[case["op"]](case, int(seed), torch.device("cuda"))
    s["case"] = dict(case)
    return s


# ---------------------------------------------------------------------------
# the plain forms
# ---------------------------------------------------------------------------

def _plain_plan(s):
    P, cap, table = s["case"]["page"], s["cap"], s["table"]
    cached, fresh = s["cached"].long(), s["fresh"].long()
    have = (cached + P - 1) // P
    need = (cached + fresh + P - 1) // P - have
    starts = torch.cat([torch.zeros_like(fresh[:1]), torch.cumsum(fresh, 0)])
    taken = torch.cumsum(need, 0) - need
    col = torch.arange(table.shape[1], device=table.device)[None, :] - have[:, None]
    new = (col >= 0) & (col < need[:, None])
    at = (taken[:, None] + col).clamp(0, s["free"].numel() - 1)
    table.copy_(torch.where(new, s["free"][at], table))
    t = torch.arange(cap, device=table.device)
    real = t < starts[-1]
    req = torch.searchsorted(starts[1:], t, right=True).clamp(max=fresh.numel() - 1)
    pos = cached[req] + t - starts[req]
    page = table[req, (pos // P).clamp(0, table.shape[1] - 1)].long()
    s["lens"].copy_(cached + fresh)
    s["starts"].copy_(starts)
    s["slots"].copy_(torch.where(real, page * P + pos % P, -1))
    s["positions"].copy_(torch.where(real, pos, 0))
    s["token_req"].copy_(torch.where(real, req, -1))
    zero = torch.zeros_like(starts[-1])
    s["info"].copy_(torch.stack([zero, starts[-1], need.sum(), zero]))
    return _plan_out(s)


def _plan_out(s):
    return {n: s[n] for n in ("table", "lens", "starts", "slots", "positions", "token_req", "info")}


def _rotate(x, cos, sin, rot, layout):
    """x [T][heads][hd] in 32 bits; cos, sin [T][1][rot / 2]."""
    y = x.clone()
    r = x[..., :rot]
    if layout == "interleaved":
        a, b = r[..., 0::2], r[..., 1::2]
        y[..., :rot] = torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2)
    else:
        a, b = r[..., :rot // 2], r[..., rot // 2:]
        y[..., :rot] = torch.cat([a * cos - b * sin, a * sin + b * cos], -1)
    return y


def _plain_rope(s):
    c = s["case"]
    angle = s["positions"].double()[:, None] * s["freqs"][None, :]  # far positions lose their angle in 32 bits
    cos, sin = ((f(angle) * s["scale"]).float()[:, None, :] for f in (torch.cos, torch.sin))
    s["q_out"].copy_(_rotate(s["q"].float(), cos, sin, c["rot"], c["layout"]))
    k = _rotate(s["k"].float(), cos, sin, c["rot"], c["layout"])
    real = torch.nonzero(s["slots"] >= 0)[:, 0]
    kc, vc = s["cache"].view(2, -1, c["nkv"], c["hd"])
    kc[s["slots"][real]] = k[real].to(kc.dtype)
    vc[s["slots"][real]] = s["v"][real].to(vc.dtype)
    return {"q": s["q_out"], "cache": s["cache"]}


def _plain_attn(s):
    c = s["case"]
    B, nh, nkv, hd, P, L = c["batch"], c["nh"], c["nkv"], c["hd"], c["page"], s["max_len"]
    j = torch.arange(L, device=s["q"].device)
    slot = s["table"][:, j // P].long().clamp(min=0) * P + j % P  # [B][L]
    kc, vc = s["cache"].view(2, -1, nkv, hd)
    q = s["q"].float().view(B, nkv, nh // nkv, hd)
    sc = torch.matmul(q, kc[slot].float().permute(0, 2, 3, 1)) * hd ** -0.5  # [B][nkv][group][L]
    if c["softcap"]:
        sc = c["softcap"] * torch.tanh(sc / c["softcap"])
    n = s["lens"].long()[:, None]
    if c["alibi"]:
        sc = sc + s["slopes"].view(1, nkv, -1, 1) * (j[None, :] - (n - 1)).float()[:, None, None, :]
    seen = j[None, :] < n
    if c["window"]:
        seen = seen & (j[None, :] >= n - c["window"])
    sc = sc.masked_fill(~seen[:, None, None, :], -math.inf)
    m = sc.amax(-1, keepdim=True)
    p = torch.exp(sc - m)
    z = p.sum(-1, keepdim=True)
    s["out"].copy_((torch.matmul(p, vc[slot].float().permute(0, 2, 1, 3)) / z).view(B, nh, hd))
    s["lse"].copy_((m + torch.log(z)).view(B, nh))
    return {"out": s["out"], "lse": s["lse"]}


def _plain_logp(s):
    c = s["case"]
    x = s["x"][:, :c["n"]].float()
    m = x.amax(-1, keepdim=True)
    d = x - m
    e = torch.exp(d)
    z = e.sum(-1, keepdim=True)
    log_z = torch.log(z)
    s["logprob"].copy_(torch.gather(d, 1, s["ids"].long()) - log_z)
    s["entropy"].copy_((log_z - torch.where(e > 0, e * d, 0.0).sum(-1, keepdim=True) / z)[:, 0])
    if c["k"]:
        # a whole number whose order is (value down, index up), so that ties go to the lowest index
        bits = (x + 0.0).view(torch.int32)
        bits = torch.where(bits >= 0, bits, bits ^ 0x7FFFFFFF).long()
        key = (bits << 32) | (0x7FFFFFFF - torch.arange(c["n"], device=x.device))
        top = torch.topk(key, c["k"], dim=1).values
        ids = 0x7FFFFFFF - (top & 0xFFFFFFFF)
        s["top_ids"].copy_(ids)
        s["top_logprob"].copy_(torch.gather(d, 1, ids) - log_z)
    return _logp_out(s)


def _logp_out(s):
    return {n: s[n] for n in ("logprob", "entropy", "top_ids", "top_logprob")}


_PLAIN = {"plan": _plain_plan, "rope_append": _plain_rope, "attention_paged": _plain_attn, "logprobs": _plain_logp}


# ---------------------------------------------------------------------------
# the framework's entry points
# ---------------------------------------------------------------------------

def _lib():
    path = os.path.join(_ROOT, "ai-agent-framework_b200")
    if path not in sys.path:
        sys.path.insert(0, path)
    import b2decode
    return b2decode


def _own_plan(s, b2):
    t = s["table"]
    b2.page_plan(s["cached"].data_ptr(), s["fresh"].data_ptr(), t.shape[0], s["case"]["page"], s["free"].data_ptr(),
                 s["n_free"].data_ptr(), t.data_ptr(), t.stride(0), t.shape[1], s["lens"].data_ptr(),
                 s["starts"].data_ptr(), s["slots"].data_ptr(), s["positions"].data_ptr(), s["token_req"].data_ptr(),
                 s["cap"], s["info"].data_ptr(), torch.cuda.current_stream().cuda_stream)
    return _plan_out(s)


def _kv(s, b2):
    """The cache's description, made once as a server makes it."""
    if "kv" not in s:
        k, v = s["cache"]
        s["kv"] = b2.paged_kv(k.data_ptr(), v.data_ptr(), _ID[s["case"]["cache"]], *k.shape)
    return s["kv"]


def _own_rope(s, b2):
    c = s["case"]
    if "rows" not in s:
        s["rows"] = b2.rope_rows(_ID[c["dtype"]], c["nh"], c["nkv"], c["hd"], c["rot"],
                                 b2.ROPE_INTERLEAVED if c["layout"] == "interleaved" else b2.ROPE_HALF,
                                 scale=s["scale"], q_stride=s["q"].stride(0), k_stride=s["k"].stride(0),
                                 v_stride=s["v"].stride(0))
    b2.rope_append(s["rows"], _kv(s, b2), s["freqs"].data_ptr(), s["positions"].data_ptr(), s["slots"].data_ptr(),
                   c["tokens"], s["q"].data_ptr(), s["k"].data_ptr(), s["v"].data_ptr(), s["q_out"].data_ptr(),
                   torch.cuda.current_stream().cuda_stream)
    return {"q": s["q_out"], "cache": s["cache"]}


def _own_attn(s, b2):
    c = s["case"]
    if "opts" not in s:
        s["opts"] = b2.paged_attn_opts(_ID[c["dtype"]], c["nh"], s["table"].shape[0], s["table"].shape[1],
                                       softcap=c["softcap"], window=c["window"],
                                       slopes=s["slopes"].data_ptr() if c["alibi"] else 0)
        s["scratch"] = torch.empty(b2.attention_paged_scratch_bytes(c["batch"], c["nh"], c["nkv"], c["hd"]),
                                   device=s["q"].device, dtype=torch.uint8)
    b2.attention_paged(_kv(s, b2), s["opts"], s["q"].data_ptr(), s["table"].data_ptr(), s["lens"].data_ptr(), 0,
                       c["batch"], s["out"].data_ptr(), s["lse"].data_ptr(), s["scratch"].data_ptr(),
                       torch.cuda.current_stream().cuda_stream)
    return {"out": s["out"], "lse": s["lse"]}


def _own_logp(s, b2):
    c, x = s["case"], s["x"]
    b2.logprobs(x.data_ptr(), _ID[c["dtype"]], c["n"], c["rows"], x.stride(0), s["ids"].data_ptr(), c["m"],
                s["logprob"].data_ptr(), s["entropy"].data_ptr(), c["k"], s["top_ids"].data_ptr(),
                s["top_logprob"].data_ptr(), torch.cuda.current_stream().cuda_stream)
    return _logp_out(s)


_OWN = {"plan": _own_plan, "rope_append": _own_rope, "attention_paged": _own_attn, "logprobs": _own_logp}


def run(state):
    op = state["case"]["op"]
    if own:
        return _OWN[op](state, _lib())
    return _PLAIN[op](state)


# ---------------------------------------------------------------------------
# work of one pass: each input read once, each output written once
# ---------------------------------------------------------------------------

_SIZE = {"f32": 4, "f16": 2, "bf16": 2}


def work(case):
    op = case["op"]
    if op == "plan":
        R, T = case["n_req"], case["tokens"]
        taken = T / case["page"] if T != R else R / case["page"]  # pages taken, on average
        return {"bytes": 12 * R + 8 * taken + 16 * (T + 5) + 8 * R + 20, "flops": 0}
    if op == "rope_append":
        T, nh, nkv, hd, rot = case["tokens"], case["nh"], case["nkv"], case["hd"], case["rot"]
        e, c = _SIZE[case["dtype"]], _SIZE[case["cache"]]
        return {"bytes": T * ((2 * nh + 2 * nkv) * hd * e + 2 * nkv * hd * c + 12) + 8 * (rot // 2),
                "flops": 3 * T * (nh + nkv) * rot}
    if op == "attention_paged":
        seen = sum(min(n, case["window"] or n) for n in _lens(case))
        nh, nkv, hd, B = case["nh"], case["nkv"], case["hd"], case["batch"]
        return {"bytes": 2 * seen * nkv * hd * 2 + 2 * B * nh * hd * _SIZE[case["dtype"]] + 4 * B * nh
                + 4 * (seen / case["page"] + B), "flops": 4 * seen * nh * hd}
    rows, n = case["rows"], case["n"]
    return {"bytes": rows * (n * _SIZE[case["dtype"]] + 8 * case["m"] + 4 + 8 * case["k"]), "flops": 5 * rows * n}


# ---------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------

def _exact_rope(case, s):
    T, hd, rot, half = case["tokens"], case["hd"], case["rot"], case["rot"] // 2
    if T * hd * (case["nh"] + 2 * case["nkv"]) > 1 << 29:
        return None
    d = torch.arange(hd, device=s["q"].device)
    if case["layout"] == "interleaved":
        pair, mate = d // 2, d ^ 1
        sign = torch.where(d % 2 == 0, -1.0, 1.0).double()
    else:
        pair, mate = d % half if half else d, torch.where(d < half, d + half, d - half)
        sign = torch.where(d < half, -1.0, 1.0).double()
    inside = d < rot
    turn = s["positions"].double().outer(s["freqs"][torch.where(inside, pair, 0)])
    cos = torch.where(inside, turn.cos() * s["scale"], 1.0)[:, None, :]
    sin = torch.where(inside, turn.sin() * s["scale"] * sign, 0.0)[:, None, :]
    mate = torch.where(inside, mate, d)

    def rotated(x):
        x = x.double()
        return x * cos + x[..., mate] * sin

    cache = s["cache"].double()
    flat = cache.view(2, -1, case["nkv"], hd)
    real = s["slots"] >= 0
    flat[0][s["slots"][real]] = rotated(s["k"])[real]
    flat[1][s["slots"][real]] = s["v"].double()[real]
    return {"q": rotated(s["q"]), "cache": cache}


def _exact_attn(case, s):
    nh, nkv, hd, P = case["nh"], case["nkv"], case["hd"], case["page"]
    out, lse = [], []
    for b, n in enumerate(s["lens"].tolist()):
        first = max(0, n - case["window"]) if case["window"] else 0
        pages = s["table"][b, first // P:(n + P - 1) // P].long()
        k, v = (c[pages].reshape(-1, nkv, hd)[first % P:first % P + n - first].double().repeat_interleave(nh // nkv, 1)
                for c in s["cache"])
        sc = torch.einsum("hd,lhd->hl", s["q"][b].double(), k) / math.sqrt(hd)
        if case["softcap"]:
            sc = torch.tanh(sc / case["softcap"]) * case["softcap"]
        if case["alibi"]:
            sc = sc - s["slopes"].double()[:, None] * torch.arange(n - first - 1, -1, -1, device=sc.device)
        z = torch.logsumexp(sc, 1)
        out.append(torch.einsum("hl,lhd->hd", torch.exp(sc - z[:, None]), v))
        lse.append(z)
    return {"out": torch.stack(out), "lse": torch.stack(lse)}


def _exact_logp(case, s):
    k, parts = case["k"], []
    for at in range(0, case["rows"], 128):
        x = s["x"][at:at + 128, :case["n"]].double()
        lp = x - torch.logsumexp(x, 1, keepdim=True)
        given = torch.gather(lp, 1, s["ids"][at:at + 128].long())
        entropy = -torch.where(torch.isfinite(lp), lp.exp() * lp, 0.0).sum(1)
        best, ids = torch.sort(x, dim=1, descending=True, stable=True)
        parts.append((given, entropy, ids[:, :k].to(torch.int32), torch.gather(lp, 1, ids[:, :k])))
    return dict(zip(("logprob", "entropy", "top_ids", "top_logprob"), (torch.cat(p) for p in zip(*parts))))


def exact(case, seed):
    if case["op"] == "plan":
        return None
    return {"rope_append": _exact_rope, "attention_paged": _exact_attn,
            "logprobs": _exact_logp}[case["op"]](case, prepare(case, seed))
