"""Cases of drafted decoding: attention for trees of drafted tokens over a paged
cache, and the verification of the drafts against the target's probabilities.

Operators, in the plain form (``own`` false) and through the framework's calls:

  tree      attention of each request's drafted tokens (its nodes, whose K/V rows
            are the last positions of the request) over the request's pages: a
            node sees every position before the nodes, and of the nodes those
            that its mask names (itself and the drafts it continues).  The cache
            is bfloat16, or 8 bits: float8_e4m3fn codes with one power-of-two
            scale per (page, kv-head) for K and one for V
  verify    which drafts the target accepts, from given random numbers, and the
            token it adds behind the last accepted one

A tree's node 0 is the token that is already decided; node i > 0 is a draft for
the place behind its parent.  With p the target's distribution behind a node (at
the temperature) and q the one that its children were drawn from one after
another, child x is accepted with probability min(1, p(x) / q(x)); if it is not,
p becomes max(p - q, 0), normalised, for the next child.  Behind the last
accepted node the added token is drawn from what p has become there.  Children
that no distribution drew (phrases from a list) count as drawn with certainty: a
rejected one is removed from p.  At temperature 0 the most likely token (the
lowest id of equal ones) is the only one accepted, and the one added.
"""
from __future__ import annotations

import math

import torch

own = False
DEV = "cuda"


# -- the cases ---------------------------------------------------------------

def listed():
    return [
        # A phrase of the user's is checked in one step on a short typed prefix.
        {"name": "tree-phrase", "kind": "tree", "bits": 16, "hq": 8, "hkv": 2, "d": 96,
         "requests": 1, "nodes": 8, "kids": 1, "cached": 24, "ragged": 0, "scattered": False},
        # A keystroke's drafts behind a long document.
        {"name": "tree-document", "kind": "tree", "bits": 16, "hq": 16, "hkv": 8, "d": 128,
         "requests": 1, "nodes": 17, "kids": 2, "cached": 4093, "ragged": 0, "scattered": False},
        # Users with a tree each, of different sizes, in a worn pool.
        {"name": "tree-batch", "kind": "tree", "bits": 16, "hq": 12, "hkv": 4, "d": 64,
         "requests": 16, "nodes": 33, "kids": 3, "cached": 1501, "ragged": 29, "scattered": True},
        # The widest trees, behind documents.
        {"name": "tree-wide", "kind": "tree", "bits": 16, "hq": 32, "hkv": 8, "d": 128,
         "requests": 4, "nodes": 200, "kids": 4, "cached": 8192, "ragged": 57, "scattered": True},
        # One user's tree behind the longest context a service keeps.
        {"name": "tree8-long", "kind": "tree", "bits": 8, "hq": 32, "hkv": 8, "d": 128,
         "requests": 1, "nodes": 40, "kids": 3, "cached": 16001, "ragged": 0, "scattered": False},
        # Users with a chain of drafts each.
        {"name": "tree8-chains", "kind": "tree", "bits": 8, "hq": 16, "hkv": 8, "d": 128,
         "requests": 8, "nodes": 6, "kids": 1, "cached": 2500, "ragged": 5, "scattered": True},
        # One short chain of a small model, an odd vocabulary, fp32 logits.
        {"name": "verify-chain", "kind": "verify", "requests": 1, "nodes": 5, "kids": 1,
         "ragged": 0, "vocab": 10007, "fp32": True, "drawn": True, "temperature": 1.0},
        # Phrases of many users, without a draft model, a sharpened target.
        {"name": "verify-phrases", "kind": "verify", "requests": 24, "nodes": 11, "kids": 2,
         "ragged": 6, "vocab": 6400, "fp32": False, "drawn": False, "temperature": 0.35},
        # One user's tree of drawn drafts.
        {"name": "verify-tree", "kind": "verify", "requests": 1, "nodes": 64, "kids": 4,
         "ragged": 0, "vocab": 151936, "fp32": False, "drawn": True, "temperature": 0.8},
        # Candidates with a drawn chain each.
        {"name": "verify-candidates", "kind": "verify", "requests": 8, "nodes": 6, "kids": 1,
         "ragged": 0, "vocab": 151936, "fp32": False, "drawn": True, "temperature": 0.7},
        # Phrases checked against the most likely tokens.
        {"name": "verify-greedy", "kind": "verify", "requests": 4, "nodes": 31, "kids": 3,
         "ragged": 3, "vocab": 16384, "fp32": True, "drawn": False, "temperature": 0.0},
        # A full batch with a drawn tree each.
        {"name": "verify-batch", "kind": "verify", "requests": 32, "nodes": 16, "kids": 2,
         "ragged": 4, "vocab": 151936, "fp32": False, "drawn": True, "temperature": 1.0},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _draw(rng):
    if rng.random() < 0.55:
        hq, hkv, d = rng.choice([(12, 4, 64), (8, 2, 96), (16, 8, 128), (32, 8, 128)])
        nodes = _log(rng, 1, 256)
        return {"kind": "tree", "bits": rng.choice([8, 16]), "hq": hq, "hkv": hkv, "d": d,
                "requests": _log(rng, 1, 32), "nodes": nodes, "kids": rng.randint(1, 5),
                "cached": 0 if rng.random() < 0.1 else _log(rng, 1, 16384),
                "ragged": rng.randint(0, nodes // 2), "scattered": rng.random() < 0.5}
    nodes = _log(rng, 1, 96)
    drawn = rng.random() < 0.6
    return {"kind": "verify", "requests": _log(rng, 1, 32), "nodes": nodes,
            "kids": rng.randint(1, 4), "ragged": rng.randint(0, nodes // 2),
            "vocab": rng.choice([6400, 16384, 151936, _log(rng, 1000, 151936)]),
            "fp32": rng.random() < 0.4, "drawn": drawn,
            "temperature": rng.choice([0.35, 0.8, 1.0, 1.3] if drawn else [0.0, 0.35, 1.0])}


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


def _sizes(case):
    """Nodes of each request."""
    return [max(1, case["nodes"] - (i * 7919 % (case["ragged"] + 1)))
            for i in range(case["requests"])]


def _cached(case):
    """Positions before the nodes of each request."""
    c = case["cached"]
    return [max(0, c - (i * 4049 % (case["ragged"] + 1))) for i in range(case["requests"])]


def _parents(case, n):
    """Levels filled one after another: a chain where kids is 1."""
    return [-1] + [(i - 1) // case["kids"] for i in range(1, n)]


def _inner(case, n):
    """Nodes with children."""
    return max(1, len(set(_parents(case, n)) - {-1}))


def work(case):
    sizes = _sizes(case)
    if case["kind"] == "tree":
        hq, hkv, d = case["hq"], case["hkv"], case["d"]
        kv = [n + c for n, c in zip(sizes, _cached(case))]
        row = 2 * d + 4 if case["bits"] == 8 else 4 * d
        words = -(-max(sizes) // 64)
        return {"bytes": sum(kv) * (hkv * row + 4) + sum(sizes) * (hq * d * 4 + 8 * words),
                "flops": 4 * hq * d * sum(a * b for a, b in zip(sizes, kv))}
    # the target's rows of the nodes with children, and the rows those were drawn from
    rows = sum(_inner(case, n) for n in sizes) * (2 if case["drawn"] else 1)
    n = rows * case["vocab"]
    return {"bytes": n * (4 if case["fp32"] else 2) + sum(sizes) * 21 + case["requests"] * 16,
            "flops": 5 * n}


# -- inputs ------------------------------------------------------------------

def _rows(g, shape, spread):
    """K or V rows: normal, each row at a magnitude of its own."""
    x = torch.randn(shape, generator=g, device=DEV)
    size = torch.randn(shape[:-1], generator=g, device=DEV).mul_(spread).exp_()
    return (x * size[..., None]).to(torch.bfloat16)


def _codes(x):
    """8-bit rows and the scales they were written with."""
    x = x.float()
    m, e = torch.frexp(x.abs().amax(-1))
    e = (e - 9 + (m > 0.875)).clamp(min=-110)
    return (torch.ldexp(x, -e[..., None]).to(torch.float8_e4m3fn),
            torch.ldexp(torch.ones_like(m), e).to(torch.bfloat16))


def _signed(word):
    return word - (1 << 64) if word >> 63 else word


def _masks(case, sizes, words):
    """Bit j % 64 of word j / 64: the node sees node j of its request."""
    out = []
    for n in sizes:
        seen = []
        for i, p in enumerate(_parents(case, n)):
            seen.append((seen[p] if p >= 0 else 0) | 1 << i)
        out += [[_signed(m >> (64 * w) & (1 << 64) - 1) for w in range(words)] for m in seen]
    return torch.tensor(out, dtype=torch.int64)


def _prepare_tree(s, g):
    c = s["case"]
    hkv, d = c["hkv"], c["d"]
    sizes, cached = _sizes(c), _cached(c)
    kv = [n + k for n, k in zip(sizes, cached)]
    total = sum(kv)
    pages = total + total // 8 + 16
    ids = (torch.randperm(pages, generator=g, device=DEV) if c["scattered"]
           else torch.arange(pages, device=DEV))
    s["indices"] = ids[:total].to(torch.int32)
    k, v = _rows(g, (pages, hkv, d), 0.2), _rows(g, (pages, hkv, d), 0.7)
    if c["bits"] == 8:
        (s["k"], ks), (s["v"], vs) = _codes(k), _codes(v)
        s["scales"] = torch.stack((ks, vs), -1).transpose(0, 1).contiguous()
    else:
        s["k"], s["v"] = k, v
    s["q"] = torch.randn((sum(sizes), c["hq"], d), generator=g,
                         device=DEV).mul_(2).to(torch.bfloat16)
    s["sizes"], s["kv_lens"] = sizes, kv
    s["cu_q"] = torch.tensor([0] + sizes, device=DEV).cumsum(0).to(torch.int32)
    s["cu_k"] = torch.tensor([0] + kv, device=DEV).cumsum(0).to(torch.int32)
    s["masks"] = _masks(c, sizes, -(-max(sizes) // 64)).to(DEV)


def _prepare_verify(s, g):
    c = s["case"]
    sizes, kids, vocab = _sizes(c), c["kids"], c["vocab"]
    total = sum(sizes)
    dtype = torch.float32 if c["fp32"] else torch.bfloat16
    first = [0]
    for n in sizes:
        first.append(first[-1] + n)
    parents = [_parents(c, n) for n in sizes]
    s["sizes"] = sizes
    s["cu"] = torch.tensor(first, dtype=torch.int32, device=DEV)
    s["parents"] = torch.tensor(sum(parents, []), dtype=torch.int32, device=DEV)
    # rows from flat to peaked, as a model's are; a draft model's are close to them
    x = torch.randn((total, vocab), generator=g, device=DEV)
    x *= torch.rand((total, 1), generator=g, device=DEV).mul_(5).add_(1)
    s["logits"] = x.to(dtype)
    s["draft"] = None
    if c["drawn"]:
        x += torch.randn((total, vocab), generator=g, device=DEV).mul_(0.7)
        s["draft"] = x.to(dtype)
    s["uniforms"] = torch.rand(total, generator=g, device=DEV)
    # the nodes' tokens: drawn from the parent's row, or likely ones of it, all different
    tokens = torch.zeros(total, dtype=torch.int64, device=DEV)
    source = s["draft"] if c["drawn"] else s["logits"]
    t = c["temperature"] if c["drawn"] else 1.0
    order = None
    if not c["drawn"]:
        # some of the drafts are what the target itself would say
        noise = torch.empty((total, vocab), device=DEV).exponential_(generator=g).log_().neg_()
        order = torch.topk(source.float() / t + noise * 0.5, min(kids, vocab)).indices
    for j in range(kids):
        node = [f + i for f, n in zip(first, sizes) for i in range(1, n) if (i - 1) % kids == j]
        at = [f + (i - 1) // kids for f, n in zip(first, sizes) for i in range(1, n)
              if (i - 1) % kids == j]
        if not node:
            continue
        node, at = torch.tensor(node, device=DEV), torch.tensor(at, device=DEV)
        if order is not None:
            tokens[node] = order[at, j]
        else:
            noise = torch.empty((len(at), vocab), device=DEV)
            noise.exponential_(generator=g).log_().neg_()
            tokens[node] = (source[at].float() / t + noise).argmax(-1)
    s["tokens"] = tokens
    # the tree's shape as tables, which the plain form keeps: the children of
    # every node, one column for each place among them, and the deepest path
    table = torch.full((total, kids), -1, dtype=torch.int64)
    for f, par in zip(first, parents):
        for i, p in enumerate(par):
            if p >= 0:
                table[f + p, (i - 1) % kids] = f + i
    s["children"] = table.to(DEV)
    deepest = 0
    for par in parents:
        depth = []
        for p in par:
            depth.append(depth[p] + 1 if p >= 0 else 0)
        deepest = max(deepest, max(depth))
    s["depth"] = deepest
    s["up"] = (s["parents"].long().clamp(min=0)
               + torch.repeat_interleave(s["cu"][:-1].long(), torch.tensor(sizes, device=DEV)))


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    s = {"case": case}
    (_prepare_tree if case["kind"] == "tree" else _prepare_verify)(s, g)
    return s


# -- the plain forms ---------------------------------------------------------

def _values(s, which, table):
    """K (0) or V (1) of the rows' pages, [rows, kv-heads, positions, head size]."""
    x = s["v" if which else "k"]
    if s["case"]["bits"] == 8:
        x = x.view(torch.uint8)[table].view(torch.float8_e4m3fn).float()
        scale = s["scales"][:, table, which].permute(1, 2, 0).float()
        return (x * scale[..., None]).transpose(1, 2)
    return x[table].float().transpose(1, 2)


def _attend(s):
    c = s["case"]
    b, hkv, d = c["requests"], c["hkv"], c["d"]
    group, t, n = c["hq"] // hkv, max(s["sizes"]), max(s["kv_lens"])
    i = torch.arange(t, device=DEV)
    new = (s["cu_q"][1:] - s["cu_q"][:-1])[:, None]
    lens = (s["cu_k"][1:] - s["cu_k"][:-1])[:, None]
    pos = torch.arange(n, device=DEV)
    table = s["indices"][(s["cu_k"][:-1, None] + pos.minimum(lens - 1)).long()].long()
    # nodes as a rectangle of t a request, the request's own ones first
    at = (s["cu_q"][:-1, None] + i.minimum(new - 1)).long()
    q = s["q"][at].float().view(b, t, hkv, group, d).permute(0, 2, 3, 1, 4)
    k, v = _values(s, 0, table), _values(s, 1, table)
    x = torch.matmul(q.reshape(b, hkv, group * t, d), k.transpose(2, 3)) * d ** -0.5
    # position p is node p - (lens - new); all that come before the nodes are seen
    node = pos - (lens - new)
    bit = node.clamp(min=0)[:, None, :].expand(-1, t, -1)
    word = s["masks"][at].gather(2, (bit // 64).clamp(max=s["masks"].shape[1] - 1))
    seen = (node < 0)[:, None, :] | ((word >> (bit % 64) & 1) == 1)
    seen &= (pos < lens)[:, None, :]
    x = x.view(b, hkv, group, t, n).masked_fill_(~seen[:, None, None], -math.inf)
    top = x.amax(-1, keepdim=True)
    x = x.sub_(torch.where(top == -math.inf, 0.0, top)).exp_()
    x = x.div_(x.sum(-1, keepdim=True).clamp(min=1e-30)).view(b, hkv, group * t, n)
    o = torch.matmul(x, v).view(b, hkv, group, t, d).permute(0, 3, 1, 2, 4)
    return o.reshape(b, t, c["hq"], d)[i < new].to(torch.bfloat16)


def _verify(s):
    c, kids, up = s["case"], s["children"], s["up"]
    tok, u = s["tokens"], s["uniforms"].double()
    total, vocab = s["logits"].shape
    root = s["cu"][:-1].long()
    node = torch.arange(total, device=DEV)
    # (64 bits: the sums over the vocabulary decide which id a number falls on)
    x = s["logits"].double()
    raw = x - torch.logsumexp(x, -1, keepdim=True)
    taken = torch.full((total,), -1, device=DEV)  # of each node, the accepted child
    if c["temperature"] == 0:
        top = x.amax(-1, keepdim=True)
        best = torch.where(x == top, torch.arange(vocab, device=DEV), vocab).amin(-1)
        for j in range(kids.shape[1]):
            child = kids[:, j]
            hit = (child >= 0) & (taken < 0) & (tok[child.clamp(min=0)] == best)
            taken = torch.where(hit, child, taken)
    else:
        p = torch.softmax(x / c["temperature"], -1)
        q = None
        if s["draft"] is not None:
            q = torch.softmax(s["draft"].double() / c["temperature"], -1)
        # what p becomes behind rejected children is max(p - lam q, 0) / mass
        lam = torch.zeros(total, dtype=torch.float64, device=DEV)
        mass = torch.ones(total, dtype=torch.float64, device=DEV)
        left = p if q is not None else p.clone()
        for j in range(kids.shape[1]):
            child = kids[:, j]
            at = child.clamp(min=0)
            here = (child >= 0) & (taken < 0)
            have = left[node, tok[at]]
            drawn = q[node, tok[at]] if q is not None else 1.0
            if q is not None:
                have = have - lam * drawn
            hit = here & (u[at] * mass * drawn < have)
            taken = torch.where(hit, child, taken)
            miss = here & ~hit
            if q is not None:
                lam = torch.where(miss, lam + mass, lam)
                rest = (p - lam[:, None] * q).clamp_(min=0).sum(-1)
                mass = torch.where(miss, rest, mass)
            else:
                mass = torch.where(miss, mass - have, mass)
                left[node, tok[at]] = torch.where(miss, 0.0, left[node, tok[at]])
    accepted = torch.zeros(total, dtype=torch.bool, device=DEV)
    accepted[root] = True
    last = root
    counts = torch.zeros(len(root), dtype=torch.int32, device=DEV)
    for _ in range(s["depth"]):
        step = taken[last]
        counts += step >= 0
        last = torch.where(step >= 0, step, last)
        accepted[last] = True
    if c["temperature"] == 0:
        pick = best[last]
    else:
        w = left[last]
        if q is not None:
            w = (w - lam[last, None] * q[last]).clamp_(min=0)
        w = torch.where(w.sum(-1, keepdim=True) > 0, w, p[last])
        cdf = w.cumsum(-1)
        pick = (cdf <= u[root, None] * w.sum(-1, keepdim=True)).sum(-1)
        pick = pick.minimum(vocab - 1 - (w > 0).flip(-1).int().argmax(-1))
    logprobs = raw[up, tok]
    logprobs[root] = raw[last, pick]
    return {"accepted": accepted, "counts": counts, "last": (last - root).int(), "next": pick,
            "logprobs": logprobs.float()}


# -- the framework's calls ---------------------------------------------------

def _own(s):
    from aios_amd import paged
    from aios_amd.sample import verify_drafts

    c = s["case"]
    if c["kind"] == "verify":
        r = verify_drafts(s["logits"], s["tokens"], s["parents"], s["cu"], s["uniforms"],
                          draft_logits=s["draft"], temperature=c["temperature"])
        return {"accepted": r.accepted, "counts": r.counts, "last": r.last,
                "next": r.next_tokens, "logprobs": r.logprobs}
    if "plan" not in s:  # the batch's schedule, which a program keeps for all layers
        s["plan"] = paged.plan("tree", s["cu_q"].cpu(), s["cu_k"].cpu(), c["hq"], c["hkv"], c["d"],
                               kv_bits=c["bits"])
    if c["bits"] == 8:
        return {"out": paged.tree_attention8(s["plan"], s["q"], s["k"], s["v"], s["scales"],
                                             s["indices"], s["cu_q"], s["cu_k"], s["masks"])}
    return {"out": paged.tree_attention(s["plan"], s["q"], s["k"], s["v"], s["indices"],
                                        s["cu_q"], s["cu_k"], s["masks"])}


def run(s):
    if own:
        return _own(s)
    return {"out": _attend(s)} if s["case"]["kind"] == "tree" else _verify(s)


# -- the definition in 64 bits -----------------------------------------------

def _exact_tree(s):
    c = s["case"]
    group = c["hq"] // c["hkv"]
    out = torch.empty(s["q"].shape, dtype=torch.float64, device=DEV)
    f = e = 0
    for n, kv in zip(s["sizes"], s["kv_lens"]):
        pages = s["indices"][e:e + kv].long()
        seen = torch.ones((n, kv), dtype=torch.bool)
        for i, p in enumerate(_parents(c, n)):
            seen[i, kv - n:] = False if p < 0 else seen[p, kv - n:]
            seen[i, kv - n + i] = True
        hidden = ~seen.to(DEV)
        for h in range(c["hkv"]):
            if c["bits"] == 8:
                k = s["k"].view(torch.uint8)[pages, h].view(torch.float8_e4m3fn).double()
                v = s["v"].view(torch.uint8)[pages, h].view(torch.float8_e4m3fn).double()
                k *= s["scales"][h, pages, 0].double()[:, None]
                v *= s["scales"][h, pages, 1].double()[:, None]
            else:
                k, v = s["k"][pages, h].double(), s["v"][pages, h].double()
            for x in range(h * group, (h + 1) * group):
                score = s["q"][f:f + n, x].double() @ k.T / math.sqrt(c["d"])
                out[f:f + n, x] = torch.softmax(score.masked_fill_(hidden, -math.inf), -1) @ v
        f, e = f + n, e + kv
    return {"out": out}


def _exact_verify(s):
    c, t = s["case"], s["case"]["temperature"]
    tok, u = s["tokens"].tolist(), s["uniforms"].double().tolist()
    raw = torch.empty(len(tok), dtype=torch.float64, device=DEV)
    f = 0
    for n in s["sizes"]:
        par = _parents(c, n)
        rows = {}

        def row(i):
            if i not in rows:
                rows[i] = torch.log_softmax(s["logits"][f + i].double(), -1)
            return rows[i]

        for i in range(1, n):
            raw[f + i] = row(par[i])[tok[f + i]]
        v = 0
        while True:
            if t == 0:
                pick = int((row(v) == row(v).amax()).nonzero()[0])
                go = [i for i in range(1, n) if par[i] == v and tok[f + i] == pick]
            else:
                p = torch.softmax(s["logits"][f + v].double() / t, -1)
                whole, go = p, []
                for i in range(1, n):
                    if par[i] != v:
                        continue
                    if s["draft"] is None:
                        q = torch.zeros_like(p)
                        q[tok[f + i]] = 1
                    else:
                        q = torch.softmax(s["draft"][f + v].double() / t, -1)
                    x = tok[f + i]
                    if u[f + i] * float(q[x]) < float(p[x]):
                        go = [i]
                        break
                    p = torch.relu(p - q)
                    p = p / p.sum() if float(p.sum()) > 0 else whole
            if not go:
                break
            v = go[0]
        if t != 0:
            over = (p.cumsum(0) > u[f] * float(p.sum())).nonzero()
            pick = int(over[0]) if len(over) else int(p.nonzero()[-1])
        raw[f] = row(v)[pick]
        f += n
    # whole numbers come from comparisons and have no nearer value
    return {"accepted": None, "counts": None, "last": None, "next": None, "logprobs": raw}


def exact(case, seed):
    s = prepare(case, seed)
    return _exact_tree(s) if case["kind"] == "tree" else _exact_verify(s)
