"""Cases of the 8-bit KV cache and of token scoring.

Operators, in the plain form (``own`` false) and through the framework's calls:

  append    K/V rows into a paged cache of float8_e4m3fn values with one
            power-of-two scale per (page, kv-head) for K and one for V
  decode    a decode step's attention over that cache: the new token's rows
            appended, then one query token per row against the row's pages
            (rows may share their first pages)
  prefill   causal attention of several new tokens per request over that cache
  score     log probabilities of given tokens, the entropy of each row and its
            most likely alternatives, from rows of logits

The cache of one layer is k8, v8 [pages, kv-heads, head size] and scales
[kv-heads, pages, 2] (bf16; K's scale, then V's).  A row's scale is 2^e with
the smallest e >= -110 that brings its largest magnitude to at most 448, and
its codes are the row divided by that, rounded to the nearest e4m3 value.
"""
from __future__ import annotations

import math

import torch

own = False
DEV = "cuda"
E_MIN = -110


# -- the cases ---------------------------------------------------------------

def listed():
    return [
        # A decode step of a small model stores one token for each of 8 candidates.
        {"name": "append-step", "kind": "append", "hkv": 2, "d": 96, "tokens": 8, "scattered": True},
        # A long document is stored, one layer at a time, into a worn pool.
        {"name": "append-prompt", "kind": "append", "hkv": 8, "d": 128, "tokens": 4096,
         "scattered": True},
        # The smallest attention step: 8 candidates on a short typed prefix.
        {"name": "decode-short", "kind": "decode", "hq": 8, "hkv": 2, "d": 96, "rows": 8,
         "prefix": 24, "own": 16, "ragged": 5, "scattered": False},
        # Candidates over a long document: their prefix is shared.
        {"name": "decode-group", "kind": "decode", "hq": 32, "hkv": 8, "d": 128, "rows": 24,
         "prefix": 4096, "own": 64, "ragged": 0, "scattered": False},
        # Users with a document each, of different lengths, in a worn pool.
        {"name": "decode-documents", "kind": "decode", "hq": 32, "hkv": 8, "d": 128, "rows": 16,
         "prefix": 0, "own": 8192, "ragged": 3001, "scattered": True},
        # One user with the longest context a service keeps.
        {"name": "decode-alone", "kind": "decode", "hq": 16, "hkv": 8, "d": 128, "rows": 1,
         "prefix": 0, "own": 16001, "ragged": 0, "scattered": False},
        # A keystroke adds a few tokens to a long cached document.
        {"name": "extend-key", "kind": "prefill", "hq": 32, "hkv": 8, "d": 128, "requests": 1,
         "new": 6, "cached": 4093, "ragged": 0},
        # A long document is read for the first time.
        {"name": "prefill-document", "kind": "prefill", "hq": 32, "hkv": 8, "d": 128,
         "requests": 1, "new": 4096, "cached": 0, "ragged": 0},
        # A batch of prompts of different lengths, some on cached prefixes.
        {"name": "prefill-batch", "kind": "prefill", "hq": 12, "hkv": 4, "d": 64, "requests": 7,
         "new": 301, "cached": 517, "ragged": 97},
        # A short continuation is scored, fp32 logits of an odd vocabulary.
        {"name": "score-few", "kind": "score", "rows": 5, "vocab": 10007, "fp32": True, "top": 8},
        # One token of each of 24 candidates, with alternatives to show.
        {"name": "score-group", "kind": "score", "rows": 24, "vocab": 151936, "fp32": False,
         "top": 5},
        # Every token of a document: its likelihood under the model.
        {"name": "score-document", "kind": "score", "rows": 2048, "vocab": 151936, "fp32": False,
         "top": 1},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _draw(rng):
    kind = rng.choice(["append", "decode", "decode", "decode", "prefill", "prefill", "score",
                       "score"])
    hq, hkv, d = rng.choice([(12, 4, 64), (8, 2, 96), (16, 8, 128), (32, 8, 128)])
    if kind == "append":
        return {"kind": kind, "hkv": hkv, "d": d, "tokens": _log(rng, 1, 4096),
                "scattered": rng.random() < 0.5}
    if kind == "decode":
        shared = rng.random() < 0.6
        length = _log(rng, 1, 128) if shared else _log(rng, 1, 16384)
        return {"kind": kind, "hq": hq, "hkv": hkv, "d": d, "rows": _log(rng, 1, 64),
                "prefix": _log(rng, 8, 16384) if shared else 0, "own": length,
                "ragged": rng.randint(0, length // 2), "scattered": rng.random() < 0.5}
    if kind == "prefill":
        new = _log(rng, 1, 4096)
        return {"kind": kind, "hq": hq, "hkv": hkv, "d": d, "requests": _log(rng, 1, 16),
                "new": new, "cached": 0 if rng.random() < 0.3 else _log(rng, 1, 12000),
                "ragged": rng.randint(0, new // 2)}
    return {"kind": kind, "rows": _log(rng, 1, 4096),
            "vocab": rng.choice([6400, 16384, 151936, _log(rng, 1000, 151936)]),
            "fp32": rng.random() < 0.4, "top": rng.choice([0, 1, 3, 5, 8, 20])}


def draw(rng):
    most = {}
    for c in listed():
        w = work(c)
        for k in w:
            most[c["kind"], k] = max(most.get((c["kind"], k), 0), w[k])
    while True:
        c = _draw(rng)
        w = work(c)
        if all(w[k] <= most[c["kind"], k] for k in w):
            return c


def _lengths(case):
    """KV length of each decode row, or (new, cached) of each request."""
    r = case["ragged"]
    if case["kind"] == "decode":
        n = [case["own"] - (i * 7919 % (r + 1)) for i in range(case["rows"])]
        return [case["prefix"] + max(1, x) for x in n]
    new = [max(1, case["new"] - (i * 7919 % (r + 1))) for i in range(case["requests"])]
    cached = [case["cached"] - (i * 4049 % (r + 1)) for i in range(case["requests"])]
    return [(a, max(0, c)) for a, c in zip(new, cached)]


def work(case):
    k = case["kind"]
    if k == "score":
        n = case["rows"] * case["vocab"]
        return {"bytes": n * (4 if case["fp32"] else 2) + case["rows"] * (16 + 12 * case["top"]),
                "flops": 5 * n}
    hkv, d = case["hkv"], case["d"]
    if k == "append":
        return {"bytes": case["tokens"] * (hkv * (6 * d + 4) + 4), "flops": case["tokens"] * hkv * 4 * d}
    lens = _lengths(case)
    if k == "decode":
        unique = case["prefix"] + sum(n - case["prefix"] for n in lens)
        return {"bytes": unique * hkv * (2 * d + 4) + 4 * sum(lens)
                + case["rows"] * d * (4 * case["hq"] + 4 * hkv),
                "flops": 4 * case["hq"] * d * sum(lens)}
    kv = sum(a + c for a, c in lens)
    return {"bytes": kv * (hkv * (2 * d + 4) + 4) + sum(a for a, _ in lens) * case["hq"] * d * 4,
            "flops": 4 * case["hq"] * d * sum(a * c + a * (a + 1) // 2 for a, c in lens)}


# -- inputs ------------------------------------------------------------------

def _rows(g, shape, spread):
    """K or V rows: normal, each row at a magnitude of its own."""
    x = torch.randn(shape, generator=g, device=DEV)
    size = torch.randn(shape[:-1], generator=g, device=DEV).mul_(spread).exp_()
    return (x * size[..., None]).to(torch.bfloat16)


def _cache(g, pages, hkv, d):
    k8, ks = _quantize(_rows(g, (pages, hkv, d), 0.2))
    v8, vs = _quantize(_rows(g, (pages, hkv, d), 0.7))
    return {"k8": k8, "v8": v8, "scales": torch.stack((ks, vs), -1).transpose(0, 1).contiguous()}


def _page_ids(g, n, scattered):
    pages = n + n // 8 + 16
    ids = (torch.randperm(pages, generator=g, device=DEV) if scattered
           else torch.arange(pages, device=DEV))
    return pages, ids[:n].to(torch.int32)


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    s = {"case": case}
    if case["kind"] == "score":
        x = torch.randn((case["rows"], case["vocab"]), generator=g, device=DEV,
                        dtype=torch.float32 if case["fp32"] else torch.bfloat16)
        # rows from flat to peaked, as a model's are
        s["logits"] = x.mul_(torch.rand((case["rows"], 1), generator=g, device=DEV).mul_(6).to(x.dtype))
        s["tokens"] = torch.randint(case["vocab"], (case["rows"],), generator=g, device=DEV)
        # half of the given tokens are likely ones
        s["tokens"][::2] = s["logits"][::2].argmax(-1)
        return s
    hkv, d = case["hkv"], case["d"]
    if case["kind"] == "append":
        t = case["tokens"]
        pages, s["loc"] = _page_ids(g, t, case["scattered"])
        s.update(_cache(g, pages, hkv, d))
        # K comes from the rotation, V is a view into the fused projection's rows
        s["k"] = _rows(g, (t, hkv, d), 0.2)
        qkv = _rows(g, (t, 4 * hkv, d), 0.7).view(t, 4 * hkv * d)
        s["v"] = qkv[:, 3 * hkv * d:].view(t, hkv, d)
        return s
    lens = _lengths(case)
    if case["kind"] == "decode":
        p = case["prefix"]
        tails = [n - p for n in lens]
        pages, ids = _page_ids(g, p + sum(tails), case["scattered"])
        table = [torch.cat((ids[:p], x)) for x in ids[p:].split(tails)]
        b, kv = case["rows"], lens
        s["k"], s["v"] = _rows(g, (b, hkv, d), 0.2), _rows(g, (b, hkv, d), 0.7)
        s["loc"] = torch.stack([x[-1] for x in table])
        s["q"] = torch.randn((b, case["hq"], d), generator=g, device=DEV).mul_(2).to(torch.bfloat16)
        s["new"] = [1] * b
    else:
        s["new"], kv = [a for a, _ in lens], [a + c for a, c in lens]
        pages, ids = _page_ids(g, sum(kv), False)
        table = list(ids.split(kv))
        s["q"] = torch.randn((sum(s["new"]), case["hq"], d), generator=g,
                             device=DEV).mul_(2).to(torch.bfloat16)
    s.update(_cache(g, pages, hkv, d))
    s["kv"] = kv
    s["indices"] = torch.cat(table)
    s["cu_q"] = torch.tensor([0] + s["new"], device=DEV).cumsum(0).to(torch.int32)
    s["cu_k"] = torch.tensor([0] + kv, device=DEV).cumsum(0).to(torch.int32)
    # the same page ids and lengths as rectangles
    pos = torch.arange(max(kv), device=DEV)
    n = torch.tensor(kv, device=DEV)[:, None]
    s["live"] = pos < n
    s["table"] = s["indices"][(s["cu_k"][:-1, None] + pos.minimum(n - 1)).long()].long()
    return s


# -- the plain forms ---------------------------------------------------------

def _quantize(x):
    x = x.float()
    a = x.abs().amax(-1)
    m, e = torch.frexp(a)  # a = m 2^e with 1/2 <= m < 1, and 448 = 7/8 2^9
    e = torch.where(a > 0, e - 9 + (m > 0.875), E_MIN).clamp(min=E_MIN)
    codes = torch.ldexp(x, -e[..., None]).to(torch.float8_e4m3fn)
    return codes, torch.ldexp(torch.ones_like(a), e).to(torch.bfloat16)


def _store(s):
    k8, ks = _quantize(s["k"])
    v8, vs = _quantize(s["v"])
    at = s["loc"].long()
    s["k8"].view(torch.uint8)[at] = k8.view(torch.uint8)
    s["v8"].view(torch.uint8)[at] = v8.view(torch.uint8)
    s["scales"][:, at] = torch.stack((ks, vs), -1).transpose(0, 1)


def _gather(s, which):
    """The values of the rows' pages, [rows, kv-heads, positions, head size]."""
    codes = s["k8" if which == 0 else "v8"].view(torch.uint8)[s["table"]]
    scale = s["scales"][:, s["table"], which].permute(1, 2, 0)
    return (codes.view(torch.float8_e4m3fn).float() * scale.float()[..., None]).transpose(1, 2)


def _attend(s):
    c = s["case"]
    b, hkv, d = len(s["kv"]), c["hkv"], c["d"]
    group, t = c["hq"] // hkv, max(s["new"])
    # queries as a rectangle of t tokens a row, the row's own ones first
    i = torch.arange(t, device=DEV)
    new = (s["cu_q"][1:] - s["cu_q"][:-1])[:, None]
    at = (s["cu_q"][:-1, None] + i.minimum(new - 1)).long()
    q = s["q"][at].float().view(b, t, hkv, group, d).permute(0, 2, 3, 1, 4)
    k, v = _gather(s, 0), _gather(s, 1)
    x = torch.matmul(q.reshape(b, hkv, group * t, d), k.transpose(2, 3)) * d ** -0.5
    last = (s["cu_k"][1:] - s["cu_k"][:-1])[:, None] - new + i  # of each query, the last key it sees
    seen = torch.arange(x.shape[-1], device=DEV) <= last[..., None]
    x = x.view(b, hkv, group, t, -1).masked_fill_(~seen[:, None, None], -math.inf)
    x = x.sub_(x.amax(-1, keepdim=True)).exp_()
    x = x.div_(x.sum(-1, keepdim=True)).view(b, hkv, group * t, -1)
    o = torch.matmul(x, v).view(b, hkv, group, t, d).permute(0, 3, 1, 2, 4)
    return o.reshape(b, t, c["hq"], d)[i < new].to(torch.bfloat16)


def _score(s):
    x, top = s["logits"], s["case"]["top"]
    f = x.float()
    d = f - f.amax(-1, keepdim=True)
    p = d.exp()
    z = p.double().sum(-1)
    log_z = z.log()
    lp = d.gather(1, s["tokens"][:, None])[:, 0] - log_z
    entropy = log_z - (p * d).double().sum(-1) / z
    # the most likely ids, the lower one first among equal logits
    bits = f.view(torch.int32).long()
    order = torch.where(bits < 0, -1 - (bits & 0x7fffffff), bits)
    ids = torch.arange(x.shape[1], device=DEV)
    best = torch.topk(order * 2 ** 20 + (2 ** 20 - 1 - ids), top, dim=-1).values
    best = 2 ** 20 - 1 - (best & (2 ** 20 - 1))
    alt = d.gather(1, best) - log_z[:, None]
    return {"logprob": lp.float(), "entropy": entropy.float(), "ids": best, "alternatives": alt.float()}


# -- the framework's calls ---------------------------------------------------

def _plan(s, phase):
    """The batch's schedule and workspace, which a program keeps for all layers."""
    from aios_amd import paged

    if "plan" not in s:
        c = s["case"]
        s["plan"] = paged.plan(phase, s["cu_q"].cpu(), s["cu_k"].cpu(), c["hq"], c["hkv"], c["d"],
                               shared_prefix_len=c.get("prefix", 0), kv_bits=8)
        s["ws"] = torch.empty(s["plan"].ws_bytes, dtype=torch.uint8, device=DEV)
    return s["plan"]


def _own(s):
    from aios_amd import paged
    from aios_amd.kernel import store_cache8
    from aios_amd.sample import token_logprobs

    kind = s["case"]["kind"]
    if kind == "append":
        store_cache8(s["k8"], s["v8"], s["scales"], s["loc"], s["k"], s["v"])
        return {"k8": s["k8"], "v8": s["v8"], "scales": s["scales"]}
    if kind == "decode":
        out = paged.append_decode8(_plan(s, "decode"), s["q"], s["k"], s["v"], s["loc"], s["k8"],
                                   s["v8"], s["scales"], s["indices"], s["cu_k"],
                                   workspace=s["ws"])
        return {"out": out, "k8": s["k8"], "v8": s["v8"], "scales": s["scales"]}
    if kind == "prefill":
        return {"out": paged.prefill8(_plan(s, "prefill"), s["q"], s["k8"], s["v8"], s["scales"],
                                      s["indices"], s["cu_q"], s["cu_k"])}
    r = token_logprobs(s["logits"], s["tokens"], top=s["case"]["top"])
    return {"logprob": r.logprobs, "entropy": r.entropies, "ids": r.top_ids,
            "alternatives": r.top_logprobs}


def run(s):
    if own:
        return _own(s)
    kind = s["case"]["kind"]
    if kind == "score":
        return _score(s)
    if kind != "prefill":
        _store(s)
    pool = {"k8": s["k8"], "v8": s["v8"], "scales": s["scales"]}
    if kind == "append":
        return pool
    out = {"out": _attend(s)}
    return {**out, **pool} if kind == "decode" else out


# -- the definition in 64 bits -----------------------------------------------

def _e4m3(x):
    """The nearest e4m3 value, ties to the even one: 2^-9 apart below 2^-6,
    an eighth of its power of two above."""
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6))) - 3)
    return torch.round(x / step) * step


def _exact_row(x):
    x = x.double()
    a = x.abs().amax(-1)
    e = torch.ceil(torch.log2((a / 448).clamp(min=2.0 ** (E_MIN - 1))))
    e = torch.where(a > 448 * torch.exp2(e), e + 1, e)
    e = torch.where(a <= 448 * torch.exp2(e - 1), e - 1, e).clamp(min=E_MIN)
    s = torch.exp2(e)
    return _e4m3(x / s[..., None]), s


def _exact_cache(s):
    at = s["loc"].long()
    pool = {"scales": s["scales"].double()}
    for w, (name, x) in enumerate((("k8", s["k"]), ("v8", s["v"]))):
        codes, scale = _exact_row(x)
        pool[name] = s[name].double()
        pool[name][at] = codes
        pool["scales"][:, at, w] = scale.T
    return pool


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "score":
        x = s["logits"].double()
        z = torch.logsumexp(x, -1, keepdim=True)
        lp = x - z
        alt = lp.sort(-1, descending=True).values[:, :case["top"]]
        got = lp.gather(1, s["tokens"][:, None])[:, 0]
        return {"logprob": got, "entropy": -(lp.exp() * lp).sum(-1), "ids": None, "alternatives": alt}
    if case["kind"] == "append":
        return _exact_cache(s)
    if case["kind"] == "decode":
        pool = _exact_cache(s)
    else:
        pool = {n: s[n].double() for n in ("k8", "v8", "scales")}
    out = torch.empty(s["q"].shape, dtype=torch.float64, device=DEV)
    group = case["hq"] // case["hkv"]
    cq, ck = s["cu_q"].tolist(), s["cu_k"].tolist()
    for r in range(len(ck) - 1):
        pages = s["indices"][ck[r]:ck[r + 1]].long()
        t, n = cq[r + 1] - cq[r], ck[r + 1] - ck[r]
        hidden = torch.ones((t, n), dtype=torch.bool, device=DEV).triu(n - t + 1)
        for h in range(case["hkv"]):
            k = pool["k8"][pages, h] * pool["scales"][h, pages, 0][:, None]
            v = pool["v8"][pages, h] * pool["scales"][h, pages, 1][:, None]
            q = s["q"][cq[r]:cq[r + 1], h * group:(h + 1) * group].double().transpose(0, 1)
            x = (q @ k.T / math.sqrt(case["d"])).masked_fill(hidden, -math.inf)
            out[cq[r]:cq[r + 1], h * group:(h + 1) * group] = (x.softmax(-1) @ v).transpose(0, 1)
    return {"out": out, **pool} if case["kind"] == "decode" else {"out": out}
