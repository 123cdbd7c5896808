"""Measured cases of the serving operators: rotary positions on the way into a paged key/value cache, attention over that
cache (with a prefix that the whole batch shares), and sampling of the next token.

`run` computes them in plain torch operations, or, where `own` is true, by the calls a user of the package makes.
"""
import math
import os
import random
import sys

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def _package():
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "moizmxfp4-public_b200")
    if path not in sys.path:
        sys.path.insert(0, path)
    import mxfp4
    return mxfp4


# ------------------------------------------------------------------------------------------------ cases
def _append(name, **kw):
    case = dict(op="append", tokens=1, heads=32, kv_heads=32, head_dim=128, rotary=128, interleaved=False, dtype="bf16", page=64, first=0,
                factor=1.0, scaling=1.0)
    case.update(kw)
    return dict(case, name=name) if name else case


def _attend(name, **kw):
    case = dict(op="attend", batch=1, heads=32, kv_heads=32, head_dim=128, dtype="bf16", page=64, shortest=1, longest=1, query_most=0, prefix=0,
                spare_pages=8)
    case.update(kw)
    return dict(case, name=name) if name else case


def _sample(name, **kw):
    case = dict(op="sample", rows=1, vocab=32000, dtype="bf16", mixed=False, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, spread=2.5)
    case.update(kw)
    return dict(case, name=name) if name else case


def listed():
    return [
        # one sequence generating: the call's latency between two layers
        _append("append one token", tokens=1, kv_heads=8, page=16, first=1000),
        # a decode step of a batch of 128 with 32 full heads, every sequence at its own position
        _append("append decode batch", tokens=128, page=64, first=512),
        # a long ragged prefill: pairs side by side, half of the head rotated, positions of a stretched context
        _append("append prefill", tokens=8191, heads=64, kv_heads=8, rotary=64, interleaved=True, dtype="fp16", page=128, first=900000, factor=8.0,
                scaling=1.25),
        # one sequence, a few tokens in: the smallest attention call there is
        _attend("decode one short", batch=1, kv_heads=8, page=16, shortest=37, longest=37),
        # the decode step of a batch of 128 between 512 and 640 tokens
        _attend("decode batch", batch=128, page=64, shortest=512, longest=640),
        # 64 answers to one long document: the document's keys are common, the answers' lengths are not
        _attend("decode shared prefix", batch=64, heads=64, kv_heads=8, page=32, shortest=1, longest=700, prefix=8191),
        # few sequences of a long context, in a cache of more than 2^31 elements
        _attend("decode long", batch=4, heads=64, kv_heads=8, page=128, shortest=50001, longest=65536, spare_pages=14000),
        # prompts of many lengths behind a common instruction
        _attend("prefill behind a prefix", batch=13, kv_heads=8, head_dim=64, dtype="fp16", page=16, shortest=1, longest=403, query_most=403, prefix=1999),
        # whole prompts
        _attend("prefill", batch=4, page=64, shortest=2048, longest=2048, query_most=2048),
        # one sequence's next token, usual settings
        _sample("sample one", rows=1, temperature=0.8, top_k=40, top_p=0.95),
        # a batch whose sequences each have their own settings, greedy ones among them
        _sample("sample mixed batch", rows=128, mixed=True),
        # a large batch over a large vocabulary, logits in 32 bits
        _sample("sample large", rows=257, vocab=131072, dtype="fp32", top_p=0.9),
    ]


def _spread(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))


def draw(rng):
    op = rng.choice(["append", "attend", "attend", "attend", "sample"])
    if op == "append":
        head_dim = rng.choice([32, 64, 128])
        kv_heads = rng.choice([1, 2, 8, 32])
        heads = kv_heads * rng.choice([1, 4, 8]) if kv_heads < 32 else 32
        return _append(None, tokens=_spread(rng, 1, 8191), heads=heads, kv_heads=kv_heads, head_dim=head_dim, rotary=rng.choice([head_dim, head_dim // 2]),
                       interleaved=rng.random() < 0.5, dtype=rng.choice(["bf16", "fp16"]), page=rng.choice([16, 32, 64, 128]),
                       first=_spread(rng, 1, 900000), factor=rng.choice([1.0, 4.0, 8.0]), scaling=rng.choice([1.0, 1.25]))
    if op == "sample":
        return _sample(None, rows=_spread(rng, 1, 257), vocab=_spread(rng, 1000, 131072), dtype=rng.choice(["bf16", "fp16", "fp32"]),
                       mixed=rng.random() < 0.5, temperature=rng.choice([0.6, 1.0, 1.4]), top_k=rng.choice([0, 1, 20, 500]),
                       top_p=rng.choice([1.0, 0.95, 0.5]), min_p=rng.choice([0.0, 0.02]), spread=rng.choice([1.0, 2.5, 5.0]))
    kv_heads = rng.choice([1, 2, 8, 32])
    heads = kv_heads * rng.choice([1, 4, 8]) if kv_heads < 32 else 32
    case = dict(heads=heads, kv_heads=kv_heads, head_dim=rng.choice([32, 64, 128]), dtype=rng.choice(["bf16", "fp16"]), page=rng.choice([16, 32, 64, 128]))
    if rng.random() < 0.5:      # one query token per sequence
        batch = _spread(rng, 1, 128)
        longest = _spread(rng, 1, min(65536, 200000000 // (batch * kv_heads * case["head_dim"])))
        prefix = 0 if rng.random() < 0.5 else _spread(rng, 1, 8191)
        return _attend(None, batch=batch, longest=longest, shortest=_spread(rng, 1, longest), prefix=prefix, **case)
    batch = _spread(rng, 1, 16)
    longest = _spread(rng, 1, 2048 // max(1, batch // 4))
    prefix = 0 if rng.random() < 0.5 else _spread(rng, 1, 2000)
    return _attend(None, batch=batch, longest=longest, shortest=_spread(rng, 1, longest), query_most=_spread(rng, 1, longest), prefix=prefix, **case)


# ------------------------------------------------------------------------------------------------ inputs
def _lengths(case):
    """Own keys and query tokens of every sequence: spread evenly over the case's range, so that the work is the case's."""
    n, lo, hi = case["batch"], case["shortest"], case["longest"]
    lens = [hi if n == 1 else lo + (hi - lo) * i // (n - 1) for i in range(n)]
    most = case["query_most"]
    return lens, [min(most, length) if most else 1 for length in lens]


def _pages(lens, page):
    return [-(-length // page) for length in lens]


def prepare(case, seed):
    dev = torch.device("cuda", torch.cuda.current_device())
    g = torch.Generator(device=dev).manual_seed(seed * 7919 + 17)
    host = random.Random(seed * 104729 + 5)
    dtype = _DTYPES[case["dtype"]]
    if case["op"] == "sample":
        rows, vocab = case["rows"], case["vocab"]
        s = dict(case=case, logits=(torch.randn(rows, vocab, generator=g, device=dev) * case["spread"]).to(dtype),
                 uniforms=torch.rand(rows, generator=g, device=dev))
        if case["mixed"]:
            pick = lambda values, kind: torch.tensor([host.choice(values) for _ in range(rows)], dtype=kind).to(dev)  # noqa: E731
            s.update(temperature=pick([0.0, 0.7, 1.0, 1.3], torch.float32), top_k=pick([0, 1, 40, 1000], torch.int32),
                     top_p=pick([1.0, 0.95, 0.5], torch.float32), min_p=pick([0.0, 0.05], torch.float32))
        else:
            s.update(temperature=case["temperature"], top_k=case["top_k"], top_p=case["top_p"], min_p=case["min_p"])
        return s
    heads, kv, dim, page = case["heads"], case["kv_heads"], case["head_dim"], case["page"]
    if case["op"] == "append":
        n = case["tokens"]
        pages = -(-n // page) + 3
        qkv = torch.randn(n, (heads + 2 * kv) * dim, generator=g, device=dev).to(dtype)      # what the projection in front leaves
        half = case["rotary"] // 2
        inv_freq = 10000.0 ** (-torch.arange(half, dtype=torch.float64) / half) / case["factor"]
        cache = lambda: torch.randn(pages, kv, page, dim, generator=g, device=dev).to(dtype)  # noqa: E731
        slots = torch.randperm(pages * page, generator=g, device=dev)[:n].to(torch.int64)
        positions = torch.arange(n, device=dev) + case["first"] if n > 1000 else torch.randint(0, case["first"] + 1, (n,), generator=g, device=dev)
        return dict(case=case, qkv=qkv, k_cache=cache(), v_cache=cache(), inv_freq=inv_freq.to(dev), positions=positions.to(torch.int64), slots=slots)
    lens, queries = _lengths(case)
    order = list(range(len(lens)))
    host.shuffle(order)
    lens, queries = [lens[i] for i in order], [queries[i] for i in order]
    need = _pages(lens, page)
    prefix_need = -(-case["prefix"] // page)
    total = sum(need) + prefix_need + case["spare_pages"]
    places = torch.randperm(total, generator=g, device=dev).to(torch.int32)
    table = torch.zeros(len(lens), max(need), dtype=torch.int32)
    at = torch.zeros(len(lens), max(need), dtype=torch.bool)
    for i, m in enumerate(need):
        at[i, :m] = True
    table, at = table.to(dev), at.to(dev)
    table[at] = places[:sum(need)]
    draw_cache = lambda: torch.empty(total, kv, page, dim, dtype=dtype, device=dev).normal_(generator=g)  # noqa: E731
    starts = [0]
    for m in queries:
        starts.append(starts[-1] + m)
    s = dict(case=case, q=torch.randn(starts[-1], heads, dim, generator=g, device=dev).to(dtype), k_cache=draw_cache(), v_cache=draw_cache(), table=table,
             lens=torch.tensor(lens, dtype=torch.int32).to(dev), starts=None, prefix_pages=None, prefix_len=None, most=max(queries))
    if case["query_most"]:
        s["starts"] = torch.tensor(starts, dtype=torch.int32).to(dev)
    if case["prefix"]:
        s["prefix_pages"] = places[sum(need):sum(need) + prefix_need].contiguous()
        s["prefix_len"] = torch.tensor([case["prefix"]], dtype=torch.int32).to(dev)
    return s


# ------------------------------------------------------------------------------------------------ one pass
def run(s):
    return {"append": _run_append, "attend": _run_attend, "sample": _run_sample}[s["case"]["op"]](s)


def _split_qkv(s):
    c = s["case"]
    n, dim = c["tokens"], c["head_dim"]
    a, b = c["heads"] * dim, (c["heads"] + c["kv_heads"]) * dim
    x = s["qkv"]
    return x[:, :a].view(n, c["heads"], dim), x[:, a:b].view(n, c["kv_heads"], dim), x[:, b:].view(n, c["kv_heads"], dim)


def _run_append(s):
    c = s["case"]
    q, k, v = _split_qkv(s)
    if own:
        out = _package().rope_append(q, k, v, s["k_cache"], s["v_cache"], s["positions"], s["slots"], s["inv_freq"], interleaved=c["interleaved"],
                                     scaling=c["scaling"])
        return {"q": out, "k": s["k_cache"], "v": s["v_cache"]}
    angle = (s["positions"].double()[:, None] * s["inv_freq"][None, :])[:, None, :]
    cos, sin = (angle.cos() * c["scaling"]).float(), (angle.sin() * c["scaling"]).float()

    def rotate(x):
        r = c["rotary"]
        y = x.float()
        if c["interleaved"]:
            a, b = y[..., 0:r:2], y[..., 1:r:2]
            turned = torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2)
        else:
            a, b = y[..., :r // 2], y[..., r // 2:r]
            turned = torch.cat([a * cos - b * sin, a * sin + b * cos], -1)
        return torch.cat([turned, y[..., r:]], -1).to(x.dtype)

    page, row = s["slots"] // c["page"], s["slots"] % c["page"]
    s["k_cache"][page, :, row] = rotate(k)
    s["v_cache"][page, :, row] = v
    return {"q": rotate(q), "k": s["k_cache"], "v": s["v_cache"]}


def _run_attend(s):
    c = s["case"]
    if own:
        out, lse = _package().paged_attention(s["q"], s["k_cache"], s["v_cache"], s["table"], s["lens"], q_starts=s["starts"],
                                              prefix_pages=s["prefix_pages"], prefix_len=s["prefix_len"], return_lse=True)
        return {"out": out, "lse": lse}
    kv, dim = c["kv_heads"], c["head_dim"]
    q, lens = s["q"].float(), s["lens"].long()
    batch, group, dev = len(lens), c["heads"] // kv, q.device
    starts = s["starts"].long() if s["starts"] is not None else torch.arange(batch + 1, device=dev)
    n = starts[1:] - starts[:-1]
    i = torch.arange(s["most"], device=dev)
    there = i[None, :] < n[:, None]                                                        # [batch, most]
    padded = q[torch.where(there, starts[:-1, None] + i[None, :], 0)]                      # [batch, most, heads, dim]
    rows = padded.view(batch, s["most"], kv, group, dim).permute(0, 2, 3, 1, 4).reshape(batch, kv, group * s["most"], dim)
    gather = lambda cache, pages: cache[pages.long()].float().transpose(-3, -4).flatten(-3, -2)  # noqa: E731  [..., kv, keys, dim]
    keys, values = gather(s["k_cache"], s["table"]), gather(s["v_cache"], s["table"])
    scale = dim ** -0.5
    score = (rows @ keys.transpose(-1, -2)).view(batch, kv, group, s["most"], -1) * scale
    j = torch.arange(keys.shape[-2], device=dev)
    seen = j[None, None, :] <= (lens - n)[:, None, None] + i[None, :, None]                # [batch, most, keys]
    score = score.masked_fill(~seen[:, None, None], -math.inf)
    if c["prefix"]:
        pk, pv = gather(s["k_cache"], s["prefix_pages"])[:, :c["prefix"]], gather(s["v_cache"], s["prefix_pages"])[:, :c["prefix"]]
        first = (rows @ pk.transpose(-1, -2)).view(batch, kv, group, s["most"], -1) * scale
        score = torch.cat([first, score], -1)
    top = score.amax(-1, keepdim=True)
    weight = (score - top).exp()
    total = weight.sum(-1, keepdim=True)
    weight = (weight / total).flatten(2, 3)
    # keys behind a sequence's end are whatever the page holds: they weigh nothing
    out = weight[..., weight.shape[-1] - keys.shape[-2]:] @ values
    if c["prefix"]:
        out = out + weight[..., :c["prefix"]] @ pv
    out = out.view(batch, kv, group, s["most"], dim).permute(0, 3, 1, 2, 4).reshape(batch, s["most"], c["heads"], dim)
    lse = (top + total.log()).squeeze(-1).permute(0, 3, 1, 2).reshape(batch, s["most"], c["heads"])
    return {"out": out[there].to(s["q"].dtype), "lse": lse[there]}


def _run_sample(s):
    if own:
        token, logprob = _package().sample_tokens(s["logits"], s["uniforms"], temperature=s["temperature"], top_k=s["top_k"], top_p=s["top_p"],
                                                  min_p=s["min_p"], return_logprobs=True)
        return {"token": token, "logprob": logprob}
    # cumulative weights decide at borders: 64 bits
    logits = s["logits"].double()
    rows, vocab = logits.shape
    column = lambda v: torch.as_tensor(v, device=logits.device).double().expand(rows).unsqueeze(1)  # noqa: E731
    heat, most, mass, least = (column(s[k]) for k in ("temperature", "top_k", "top_p", "min_p"))
    x, index = logits.sort(dim=1, descending=True, stable=True)
    greedy = heat <= 0
    x = (x - x[:, :1]) / torch.where(greedy, 1.0, heat)
    weight = x.exp()
    rank = torch.arange(vocab, device=logits.device)[None, :]
    weight = torch.where((most > 0) & (rank >= most), 0.0, weight)
    before = weight.cumsum(1) - weight
    weight = torch.where((mass < 1) & (rank > 0) & (before >= mass * weight.sum(1, keepdim=True)), 0.0, weight)
    weight = torch.where((weight < least) | (greedy & (rank > 0)), 0.0, weight)
    up_to = weight.cumsum(1)
    total = up_to[:, -1:]
    at = (up_to <= s["uniforms"].double()[:, None] * total).sum(1, keepdim=True)
    return {"token": index.gather(1, at)[:, 0], "logprob": (x.gather(1, at) * ~greedy - total.log())[:, 0].float()}


# ------------------------------------------------------------------------------------------------ work
def work(case):
    size = 4 if case["dtype"] == "fp32" else 2
    if case["op"] == "append":
        moved = case["tokens"] * (case["heads"] + 2 * case["kv_heads"]) * case["head_dim"]
        return {"bytes": 2 * moved * size + 16 * case["tokens"], "flops": 3 * moved}
    if case["op"] == "sample":
        n = case["rows"] * case["vocab"]
        return {"bytes": n * size + 16 * case["rows"], "flops": 4 * n}
    lens, queries = _lengths(case)
    tokens = sum(queries)
    pairs = sum(m * case["prefix"] + m * length - m * (m - 1) // 2 for length, m in zip(lens, queries))
    keys = sum(lens) + case["prefix"]
    return {"bytes": size * case["head_dim"] * (2 * keys * case["kv_heads"] + 2 * tokens * case["heads"]) + 4 * tokens * case["heads"],
            "flops": 4 * case["head_dim"] * case["heads"] * pairs}


# ------------------------------------------------------------------------------------------------ the definitions, in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    return {"append": _exact_append, "attend": _exact_attend, "sample": _exact_sample}[case["op"]](s, case)


def _exact_append(s, c):
    q, k, v = (x.double() for x in _split_qkv(s))
    turn = torch.polar(torch.full_like(s["inv_freq"], c["scaling"]).expand(c["tokens"], -1).contiguous(),
                       s["positions"].double()[:, None] * s["inv_freq"]).unsqueeze(1)      # one complex factor per token and pair

    def rotate(x):
        r = c["rotary"]
        z = torch.view_as_complex(x[..., :r].unflatten(-1, (r // 2, 2) if c["interleaved"] else (2, r // 2)).transpose(-1, -1 if c["interleaved"] else -2).contiguous())
        y = torch.view_as_real(z * turn)
        x = x.clone()
        x[..., :r] = (y if c["interleaved"] else y.transpose(-1, -2)).flatten(-2)
        return x

    out = {"q": rotate(q), "k": s["k_cache"].double(), "v": s["v_cache"].double()}
    page, row = s["slots"].div(c["page"], rounding_mode="floor"), s["slots"].remainder(c["page"])
    out["k"].transpose(1, 2)[page, row] = rotate(k)
    out["v"].transpose(1, 2)[page, row] = v
    return out


def _exact_attend(s, c):
    """Sequence by sequence and key head by key head, over the keys that a query sees and no others."""
    kv, dim, page, prefix = c["kv_heads"], c["head_dim"], c["page"], c["prefix"]
    group = c["heads"] // kv
    lens = s["lens"].tolist()
    starts = s["starts"].tolist() if s["starts"] is not None else list(range(len(lens) + 1))
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=s["q"].device)
    lse = torch.full(s["q"].shape[:2], -math.inf, dtype=torch.float64, device=s["q"].device)
    fetch = lambda cache, pages, n, h: cache[pages.long(), h].double().reshape(-1, dim)[:n]  # noqa: E731
    for h in range(kv):
        at = slice(h * group, (h + 1) * group)
        common = [fetch(x, s["prefix_pages"], prefix, h) for x in (s["k_cache"], s["v_cache"])] if prefix else None
        for b, length in enumerate(lens):
            pages = s["table"][b, :-(-length // page)]
            k, v = fetch(s["k_cache"], pages, length, h), fetch(s["v_cache"], pages, length, h)
            if prefix:
                k, v = torch.cat([common[0], k]), torch.cat([common[1], v])
            n = starts[b + 1] - starts[b]
            x = s["q"][starts[b]:starts[b + 1], at].double()                               # [n, group, dim]
            score = torch.einsum("ngd,kd->ngk", x, k) / math.sqrt(dim)
            last = torch.arange(prefix + length - n, prefix + length, device=x.device)     # the last key each query sees
            score.masked_fill_((torch.arange(len(k), device=x.device)[None, :] > last[:, None])[:, None], -math.inf)
            lse[starts[b]:starts[b + 1], at] = score.logsumexp(-1)
            out[starts[b]:starts[b + 1], at] = torch.einsum("ngk,kd->ngd", score.softmax(-1), v)
    return {"out": out, "lse": lse}


def _exact_sample(s, c):
    """Row by row over a sorted list, as the definition reads."""
    tokens, logprobs = [], []
    settings = {k: s[k].tolist() if isinstance(s[k], torch.Tensor) else [s[k]] * c["rows"] for k in ("temperature", "top_k", "top_p", "min_p")}
    uniforms = s["uniforms"].double().tolist()
    for r in range(c["rows"]):
        row = s["logits"][r].double()
        heat, k, p, m = (settings[n][r] for n in ("temperature", "top_k", "top_p", "min_p"))
        if heat <= 0:
            tokens.append(int((row == row.max()).nonzero()[0]))
            logprobs.append(0.0)
            continue
        order = torch.argsort(-row, stable=True)
        x = (row[order] - row.max()) / heat
        if k > 0:
            x = x[:int(k)]
        w = x.exp()
        if p < 1:
            reached = (w.cumsum(0) >= p * w.sum()).nonzero()
            w = w[:int(reached[0]) + 1]
        w = w[w >= m] if m > 0 else w
        total = w.sum()
        at = min(int(torch.searchsorted(w.cumsum(0), uniforms[r] * total, right=True)), len(w) - 1)
        tokens.append(int(order[at]))
        logprobs.append(float(x[at] - total.log()))
    return {"token": torch.tensor(tokens, device=s["logits"].device), "logprob": torch.tensor(logprobs, dtype=torch.float64, device=s["logits"].device)}
