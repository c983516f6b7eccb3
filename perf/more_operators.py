"""More of what serving several requests at once takes, as cases that can be timed: a paged cache held in 8 bits (appending to it, attention over it), attention of
requests that begin alike, whose common beginning is gone through once for all of them, and drafted tokens checked against a target's distribution.

A case is a dict of plain values:
  kind      "append": spy_hip_paged_append_q8, "attend": spy_hip_paged_attention_q8, "shared": spy_hip_paged_attention_shared, "verify": spy_hip_sample_verify
  append, attend, shared:
    seqs    requests in the batch; `chunks` of them bring up to `new` new tokens, the others one
    kv      the longest request's cached tokens, its new ones included (shared: without the common ones); `ragged`: the others are shorter, else all alike
    heads, kv_heads, hd, page: query heads, K/V heads, their width, positions of a page
    type    append: type of q, k, v; attend, shared: type of the output ("f32" or "f16"); mode: 0 neighbouring pairs, 2 halves; base, freq_scale, dims: the rotation
    window  attend: 0, or how many positions back a token sees
    groups, loose, prefix, cache: shared: the last `loose` requests share nothing, the others belong to so many groups, each with up to `prefix` tokens in common;
            "f16" or "q8" pages
  verify:
    seqs, drafts, vocab: requests, drafted tokens of one at most, vocabulary; `drafter`: the drafts were drawn from logits (else looked up, no distribution)
    filters "all": temperature, top-k, top-p and min-p by row, some requests greedy; "top_p": temperature and top-p
"""
import ctypes as C
import math

import numpy as np
import torch

own = False


def listed():
    head = {"heads": 32, "kv_heads": 32, "hd": 128}
    group = {"heads": 32, "kv_heads": 8, "hd": 128}
    rope = {"base": 10000.0, "freq_scale": 1.0, "dims": 128}
    return [
        # one request, one token: the smallest call there is
        {"name": "append_q8_1", "kind": "append", "seqs": 1, "chunks": 0, "new": 1, "kv": 1001, "ragged": False, **head, "page": 64, "type": "f32", "mode": 0, **rope},
        # a prompt's chunk of the 7B shape
        {"name": "append_q8_prompt_2048", "kind": "append", "seqs": 1, "chunks": 1, "new": 2048, "kv": 2048, "ragged": False, **head, "page": 64, "type": "f32", "mode": 0, **rope},
        # the token loop's attention at the 7B shape: one request, 4096 cached tokens
        {"name": "attend_q8_1_4096", "kind": "attend", "seqs": 1, "chunks": 0, "new": 1, "kv": 4096, "ragged": False, **head, "page": 64, "type": "f32", "window": 0},
        # a step of a full batch: what a cache of half the bytes is for
        {"name": "attend_q8_64_ragged", "kind": "attend", "seqs": 64, "chunks": 0, "new": 1, "kv": 8000, "ragged": True, **group, "page": 16, "type": "f16", "window": 0},
        # a chunk of a long document on what came before it
        {"name": "attend_q8_512_on_7680", "kind": "attend", "seqs": 1, "chunks": 1, "new": 512, "kv": 8192, "ragged": False, **group, "page": 64, "type": "f16", "window": 0},
        # a few samples of one short prompt
        {"name": "shared_4_600", "kind": "shared", "seqs": 4, "chunks": 0, "new": 1, "kv": 40, "ragged": True, "groups": 1, "loose": 0, "prefix": 600, "cache": "f16", **head, "page": 64,
         "type": "f32"},
        # a full batch behind four system prompts, some requests without one
        {"name": "shared_64_8000", "kind": "shared", "seqs": 64, "chunks": 0, "new": 1, "kv": 900, "ragged": True, "groups": 4, "loose": 4, "prefix": 8000, "cache": "f16", **group, "page": 16,
         "type": "f16"},
        # questions about one long document, in 8 bits
        {"name": "shared_q8_32_20000", "kind": "shared", "seqs": 32, "chunks": 0, "new": 1, "kv": 500, "ragged": True, "groups": 1, "loose": 0, "prefix": 20001, "cache": "q8", **group, "page": 64,
         "type": "f16"},
        # new requests whose prompts follow the same examples
        {"name": "shared_prompts_2000", "kind": "shared", "seqs": 8, "chunks": 8, "new": 201, "kv": 201, "ragged": True, "groups": 1, "loose": 0, "prefix": 2000, "cache": "f16", **head, "page": 32,
         "type": "f16"},
        # one request with four tokens of a small model: the step that is to take less time than four
        {"name": "verify_1_32000", "kind": "verify", "seqs": 1, "drafts": 4, "vocab": 32000, "drafter": True, "filters": "all"},
        # a batch of requests with settings of their own
        {"name": "verify_32_32000", "kind": "verify", "seqs": 32, "drafts": 5, "vocab": 32000, "drafter": True, "filters": "all"},
        # a large batch whose drafts were looked up in the prompts, a large vocabulary of odd size
        {"name": "verify_64_100003", "kind": "verify", "seqs": 64, "drafts": 3, "vocab": 100003, "drafter": False, "filters": "top_p"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))


def draw(rng):
    kind = rng.choice(["append", "attend", "attend", "shared", "shared", "verify"])
    if kind == "verify":
        vocab, drafter = _log(rng, 1000, 131072), rng.random() < 0.6
        rows = 256 * 100003 // vocab // (2 if drafter else 1)
        drafts = min(rng.randint(1, 8), max(1, rows - 1))
        return {"kind": kind, "seqs": max(1, min(_log(rng, 1, 64), rows // (drafts + 1))), "drafts": drafts, "vocab": vocab, "drafter": drafter, "filters": rng.choice(["all", "top_p"])}
    heads, kv_heads = rng.choice([(32, 32), (32, 8), (24, 8), (16, 1), (10, 2), (8, 8), (64, 8)])
    shape = {"heads": heads, "kv_heads": kv_heads, "hd": rng.choice([64, 128, 128, 256]), "page": rng.choice([16, 32, 64, 128, 256])}
    if kind == "append":
        new = rng.choice([1, _log(rng, 2, 700)])
        seqs = _log(rng, 1, 64) if new == 1 else min(_log(rng, 1, 8), max(1, 1500 // new))
        return {"kind": kind, "seqs": seqs, "chunks": 0 if new == 1 else rng.randint(1, seqs), "new": new, "kv": new + _log(rng, 1, 20000), "ragged": rng.random() < 0.5, **shape,
                "dims": shape["hd"] // rng.choice([1, 1, 2]), "type": rng.choice(["f32", "f16"]), "mode": rng.choice([0, 2]), "base": rng.choice([10000.0, 500000.0]),
                "freq_scale": rng.choice([1.0, 0.25])}
    shape["hd"] = min(shape["hd"], 128) if kv_heads == 32 or heads == 64 else shape["hd"]
    wide = kv_heads * shape["hd"] / 1024
    if rng.random() < 0.6:
        seqs, new, chunks = _log(rng, 1 if kind == "attend" else 2, 64), 1, 0
    else:
        seqs, new = _log(rng, 1 if kind == "attend" else 2, 16), _log(rng, 2, 600)
        chunks = rng.randint(1, seqs)
    most = min(30000, 300000 / wide / seqs, 1.4e10 / (seqs * heads * new * shape["hd"]))          # cached tokens of a request
    if most < 2 * new + 32:
        new, chunks = 1, 0
        most = min(30000, 300000 / wide / seqs, 1.4e10 / (seqs * heads * shape["hd"]))
    common = {"kind": kind, "seqs": seqs, "chunks": chunks, "new": new, "ragged": rng.random() < 0.7, **shape, "type": rng.choice(["f16", "f16", "f32"])}
    if kind == "attend":
        return {**common, "kv": max(new, _log(rng, 16, most)), "window": rng.choice([0, 0, _log(rng, 16, 4096)])}
    kv = max(new, _log(rng, 1, min(2000, most / 2)))
    groups = rng.randint(1, min(6, seqs // 2))
    return {**common, "kv": kv, "groups": groups, "loose": rng.choice([0, 0, rng.randint(0, seqs - 2 * groups)]), "prefix": _log(rng, 16, max(16, most - kv)), "cache": rng.choice(["f16", "q8"])}


def _part(case, i):
    """every length between a fifth of the longest and the longest, the first one the longest"""
    return 1.0 - 0.8 * ((i * 0.6180339887) % 1.0) if case["ragged"] else 1.0


def _groups(case):
    """(first request of each group and the end of the last, tokens that each group has in common), from the case alone"""
    if case["kind"] != "shared":
        return [0], []
    n, g = case["seqs"] - case["loose"], case["groups"]
    return [n * i // g for i in range(g + 1)], [max(1, int(case["prefix"] * _part(case, i))) for i in range(g)]


def _lengths(case):
    """(new tokens, cached tokens, those of them in common with the group) of each request, from the case alone"""
    start, common = _groups(case)
    news, kvs, pre = [], [], []
    for i in range(case["seqs"]):
        new = max(1, int(case["new"] * _part(case, i))) if i < case["chunks"] else 1
        pre.append(next((common[g] for g in range(len(common)) if start[g] <= i < start[g + 1]), 0))
        news.append(new)
        kvs.append(pre[-1] + max(new, int(case["kv"] * _part(case, i))))
    return news, kvs, pre


def _visible(case):
    """pairs of a query token and a cached token that it sees, and the cached tokens that have to be read"""
    pairs = read = 0
    w = case.get("window", 0)
    for new, kv, pre in zip(*_lengths(case)):
        pairs += sum(min(p + 1, w or kv) for p in range(kv - new, kv))
        read += min(kv, w + new - 1) if w else kv - pre
    return pairs, read + sum(_groups(case)[1])


# ---- 8 bits: blocks of 32 elements of a row, d = (largest magnitude) / 127 as fp16 and q = x * 127 / (largest magnitude) to the nearest whole number, halves to even --
def _to_q8(x, dim):
    """x in 32 bits, blocks along `dim`: the whole numbers and the scales"""
    dim %= x.dim()
    b = x.unflatten(dim, (-1, 32))
    top = b.abs().amax(dim=dim + 1, keepdim=True)
    inv = torch.where(top > 0, 127.0 / top, torch.zeros_like(top))
    return torch.round(b * inv).to(torch.int8).flatten(dim, dim + 1), (top / 127.0).squeeze(dim + 1).half()


def _values(q, d, dim, out=None):
    """what the pages stand for: fp16(d * q)"""
    dim %= q.dim()
    return torch.mul(q.unflatten(dim, (-1, 32)), d.unsqueeze(dim + 1), out=out).flatten(dim, dim + 1)


def _settings(case, rows, seq, gen):
    n = case["seqs"]

    def pick(values):
        return torch.tensor(values, device="cuda")[torch.randint(0, len(values), (n,), generator=gen, device="cuda")][seq]

    p = {"temperature": (torch.rand(n, generator=gen, device="cuda") * 0.7 + 0.6)[seq], "top_p": pick([0.8, 0.9, 0.95])}
    if case["filters"] == "all":
        p["top_k"] = pick([20, 40, 50, 500, 0]).to(torch.int32)
        p["min_p"] = pick([0.0, 0.0, 0.05])
        p["top_p"] = torch.where((torch.rand(n, generator=gen, device="cuda") < 0.3)[seq], torch.ones_like(p["top_p"]), p["top_p"])
        p["temperature"] = torch.where(seq % 8 == 5, torch.zeros_like(p["temperature"]), p["temperature"])
    return p


def _drafts(case):
    return [max(1, int(case["drafts"] * (1.0 - 0.7 * ((i * 0.6180339887) % 1.0)))) for i in range(case["seqs"])]


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    randn = lambda *shape: torch.randn(shape, generator=gen, device="cuda")                     # noqa: E731
    i32 = lambda v: torch.tensor(np.asarray(v, np.int32), device="cuda")                         # noqa: E731
    s = {"case": case}
    if case["kind"] == "verify":
        n, vocab = case["seqs"], case["vocab"]
        rows_of = [d + 1 for d in _drafts(case)]
        rows = sum(rows_of)
        seq = torch.tensor(np.repeat(np.arange(n), rows_of), device="cuda")
        s.update(row_start=i32(np.concatenate([[0], np.cumsum(rows_of)])), rows=rows, param=_settings(case, rows, seq, gen))
        s["logits"] = randn(rows, vocab) * 2.5
        at = torch.randint(0, vocab, (rows, 24), generator=gen, device="cuda")                   # the tokens that a context makes likely
        s["logits"].scatter_add_(1, at, 4.0 + 5.0 * torch.rand((rows, 24), generator=gen, device="cuda"))
        draft = s["logits"] + 0.7 * randn(rows, vocab)                                            # a smaller model: much the same
        s["draft_param"] = _settings(case, rows, seq, gen)
        u = torch.rand(rows, generator=gen, device="cuda")
        if case["drafter"]:
            s["draft_logits"] = draft
            s["drafted"] = _drawn(_distribution(draft, s["draft_param"]), u).to(torch.int32)
        else:
            s["drafted"] = torch.where(u < 0.6, s["logits"].argmax(dim=1), at[:, 0]).to(torch.int32)
        s["accept"], s["param"]["uniform"] = (torch.rand(rows, generator=gen, device="cuda") for _ in range(2))
        s["tokens"] = torch.zeros(rows, dtype=torch.int32, device="cuda")
        s["accepted"] = torch.zeros(n, dtype=torch.int32, device="cuda")
        s["probs"] = torch.zeros(rows, device="cuda")
        return s
    news, kvs, pre = _lengths(case)
    H, G, hd, ps, rows = case["heads"], case["kv_heads"], case["hd"], case["page"], sum(news)
    append, q8 = case["kind"] == "append", case.get("cache", "q8") == "q8"
    start, common = _groups(case)
    leader = [next((start[g] for g in range(len(common)) if start[g] <= i < start[g + 1]), i) for i in range(len(kvs))]
    first = [(kv - new) // ps if append else p // ps if i != leader[i] else 0 for i, (new, kv, p) in enumerate(zip(news, kvs, pre))]     # an append's pages are those that it touches
    count = [(kv + ps - 1) // ps - f for kv, f in zip(kvs, first)]
    n_page, width = sum(count) + 3, max((kv + ps - 1) // ps for kv in kvs)
    order = np.random.default_rng(seed).permutation(n_page)
    table, at = np.zeros((len(kvs), width), np.int32), 0
    for i, (f, c) in enumerate(zip(first, count)):
        table[i, f:f + c] = order[at:at + c]
        at += c
        if leader[i] != i:
            table[i, :f] = table[leader[i], :f]
    s.update(row_start=i32(np.concatenate([[0], np.cumsum(news)])), kv_len=i32(kvs), table=i32(table), rows=rows, max_new=max(news), max_kv=max(kvs))
    s["k_pages"] = torch.empty((n_page, G, ps, hd), dtype=torch.float16, device="cuda").normal_(generator=gen)
    s["k_pages"] *= (1.0 + 3.0 * torch.rand(hd, generator=gen, device="cuda") ** 8).half()        # some dimensions of keys are larger than others
    s["v_pages"] = torch.empty((n_page, G, hd, ps), dtype=torch.float16, device="cuda").normal_(generator=gen)
    for i, p in enumerate(pre):                                                                    # the page in which the common tokens end is a copy of each request's own
        if leader[i] != i and p % ps:
            mine, its = int(table[i, p // ps]), int(table[leader[i], p // ps])
            s["k_pages"][mine, :, :p % ps] = s["k_pages"][its, :, :p % ps]
            s["v_pages"][mine, :, :, :p % ps] = s["v_pages"][its, :, :, :p % ps]
    if q8:
        for name, dim in (("k", -1), ("v", -2)):
            got = [_to_q8(x.float(), dim) for x in s[name + "_pages"].split(max(1, (1 << 27) // (G * ps * hd)))]
            s[name + "_pages"], s[name + "_scales"] = torch.cat([g[0] for g in got]), torch.cat([g[1] for g in got])
    if append:
        dt = torch.float32 if case["type"] == "f32" else torch.float16
        s["q"], s["k"], s["v"] = randn(rows, H, hd).to(dt), randn(rows, G, hd).to(dt), randn(rows, G, hd).to(dt)
        s["q_out"] = torch.zeros((rows, H, hd), dtype=torch.float16, device="cuda")
        for name, dim in (("k", -1), ("v", -2)):
            s[name + "_values"] = torch.empty_like(s[name + "_pages"].unflatten(dim, (-1, 32)), dtype=torch.float16)
        return s
    s["q"] = (randn(rows, H, hd) * 1.5).half()
    s["out"] = torch.zeros((rows, H, hd), dtype=torch.float32 if case["type"] == "f32" else torch.float16, device="cuda")
    if case["kind"] == "shared":
        s.update(seq_start=i32(start), common=i32(common), max_common=max(common),
                 max_rows=max(sum(news[a:b]) for a, b in zip(start, start[1:])))
    return s


# ---- the plain forms ----------------------------------------------------------------------------------------------------------------
def _sequences(s):
    """request of every row, and how many of its rows come after it"""
    row = torch.arange(s["rows"], device="cuda")
    seq = torch.searchsorted(s["row_start"][1:].long(), row, right=True)
    return seq, s["row_start"].long()[seq + 1] - 1 - row


def _rotated(x, pos, case):
    nd = case["dims"]
    i = torch.arange(nd // 2, device="cuda", dtype=torch.float64)
    angle = pos.double()[:, None] * (case["freq_scale"] * case["base"] ** (-2.0 * i / nd))        # far positions: 64 bits
    c, s = torch.cos(angle).float()[:, None, :], torch.sin(angle).float()[:, None, :]
    x = x.float()
    a, b = (x[..., 0:nd:2], x[..., 1:nd:2]) if case["mode"] == 0 else (x[..., :nd // 2], x[..., nd // 2:nd])
    u, v = a * c - b * s, a * s + b * c
    y = torch.stack([u, v], dim=-1).flatten(-2) if case["mode"] == 0 else torch.cat([u, v], dim=-1)
    return torch.cat([y, x[..., nd:]], dim=-1)


def _append(s):
    case, ps = s["case"], s["case"]["page"]
    seq, after = _sequences(s)
    pos = s["kv_len"].long()[seq] - 1 - after
    page, at = s["table"][seq, pos // ps].long(), pos % ps
    s["k_pages"][page, :, at, :], s["k_scales"][page, :, at, :] = _to_q8(_rotated(s["k"], pos, case), -1)
    s["v_pages"][page, :, :, at], s["v_scales"][page, :, :, at] = _to_q8(s["v"].float(), -1)
    return {"q": _rotated(s["q"], pos, case).half(), **_read_back(s)}


def _read_back(s):
    """the pages as the values that they stand for"""
    return {"k_pages": _values(s["k_pages"], s["k_scales"], -1, s["k_values"]), "v_pages": _values(s["v_pages"], s["v_scales"], -2, s["v_values"])}


def _attend(s):
    case, ps = s["case"], s["case"]["page"]
    H, G, hd, n = case["heads"], case["kv_heads"], case["hd"], case["seqs"]
    j = torch.arange(s["max_kv"], device="cuda")
    page, at = s["table"][:, j // ps].long(), (j % ps).expand(n, -1)
    k, v = s["k_pages"][page, :, at, :], s["v_pages"][page, :, :, at]                             # [request][position][K/V head][hd]
    if "k_scales" in s:
        k, v = _values(k, s["k_scales"][page, :, at, :], -1), _values(v, s["v_scales"][page, :, :, at], -1)
    k, v = k.permute(0, 2, 1, 3).float(), v.permute(0, 2, 1, 3).float()
    start, kv = s["row_start"].long(), s["kv_len"].long()
    i = torch.arange(s["max_new"], device="cuda")
    there = i[None, :] < (start[1:] - start[:-1])[:, None]
    row = (start[:-1, None] + i).clamp(max=s["rows"] - 1)
    q = s["q"][row].float().reshape(n, -1, G, H // G, hd).permute(0, 2, 1, 3, 4).reshape(n, G, -1, hd)
    pos = (kv - (start[1:] - start[:-1]))[:, None] + i                                            # [request][new token]
    seen = (j <= pos[..., None]) & (j < kv[:, None, None])
    if case.get("window"):
        seen &= j > pos[..., None] - case["window"]
    seen = seen.repeat_interleave(H // G, dim=1)[:, None]                                         # [request][1][token, head of the group][position]
    x = torch.matmul(q, k.transpose(2, 3)).mul_(1.0 / math.sqrt(hd)).masked_fill_(~seen, -math.inf)
    top = x.amax(dim=-1, keepdim=True)
    e = x.sub_(torch.where(top > -math.inf, top, torch.zeros_like(top))).exp_()
    total = e.sum(dim=-1, keepdim=True)
    o = torch.matmul(e, v) / torch.where(total > 0, total, torch.ones_like(total))
    o = o.reshape(n, G, -1, H // G, hd).permute(0, 2, 1, 3, 4).reshape(n, -1, H, hd)
    return o[there].to(s["out"].dtype)


def _distribution(logits, param):
    """probabilities of every row's tokens under its settings, in 64 bits: they are compared with each other and summed up to borders"""
    x = logits.double()
    y, order = torch.sort(x, dim=1, descending=True, stable=True)
    t = param["temperature"].double()[:, None]
    greedy = t <= 0
    w = torch.exp((y - y[:, :1]) / torch.where(greedy, torch.ones_like(t), t))
    rank = torch.arange(x.shape[1], device="cuda")[None]
    if "top_k" in param:
        k = param["top_k"].long()[:, None]
        w = torch.where((k > 0) & (rank >= k), torch.zeros_like(w), w)
    before = torch.cumsum(w, dim=1) - w
    p = param["top_p"].double()[:, None]
    keep = (p >= 1) | (before < p * w.sum(dim=1, keepdim=True))
    if "min_p" in param:
        keep &= w >= param["min_p"].double()[:, None]
    keep = torch.where(greedy, rank == 0, keep | (rank == 0))
    w = torch.where(keep, w, torch.zeros_like(w))
    return torch.zeros_like(w).scatter_(1, order, w / w.sum(dim=1, keepdim=True))


def _drawn(w, uniform):
    run_ = torch.cumsum(w, dim=1)
    return (run_ > uniform.double()[:, None] * run_[:, -1:]).to(torch.uint8).argmax(dim=1)


def _verify(s):
    rows, vocab = s["logits"].shape
    seq, after = _sequences(s)
    last = after == 0                                                                              # the row behind a request's drafts
    d = s["drafted"].long()[:, None]
    p = _distribution(s["logits"], s["param"])
    q = _distribution(s["draft_logits"], s["draft_param"]) if "draft_logits" in s else torch.zeros_like(p).scatter_(1, d, 1.0)
    fine = (s["accept"].double() * q.gather(1, d)[:, 0] < p.gather(1, d)[:, 0]) & ~last
    first = s["row_start"].long()
    row = torch.arange(rows, device="cuda")
    refused = torch.where(fine, torch.full_like(row, rows), row)                                   # the first row of a request whose draft is not taken; its last row at the latest
    stop = torch.full((s["case"]["seqs"],), rows, device="cuda").scatter_reduce_(0, seq, refused, "amin")
    q = torch.where(last[stop][:, None], torch.zeros_like(q[stop]), q[stop])
    left = (p[stop] - q).clamp_(min=0)
    left = torch.where(left.sum(dim=1, keepdim=True) > 0, left, p[stop])
    token = _drawn(left, s["param"]["uniform"][stop])
    out = torch.where(row < stop[seq], s["drafted"].long(), torch.where(row == stop[seq], token[seq], torch.full_like(row, -1)))
    prob = torch.where(out >= 0, p.gather(1, out.clamp(min=0)[:, None])[:, 0], torch.zeros_like(p[:, 0]))
    return {"tokens": out.to(torch.int32), "accepted": (stop - first[:-1]).to(torch.int32), "probs": prob.float()}


# ---- the framework's calls ----------------------------------------------------------------------------------------------------------
def _tensor(H, x, dims):
    t = {torch.float32: H.F32, torch.float16: H.F16, torch.int8: H.I8}[x.dtype]
    return H.tensor(x.data_ptr(), t, dims)


def _bind(s):
    """What a program that serves requests keeps beside its buffers: their descriptions and the workspace."""
    from spy_amd import _lib as H
    H.init(0)
    L, case, ref = H.load(), s["case"], lambda x: None if x is None else C.byref(x)               # noqa: E731
    if case["kind"] == "verify":
        at = lambda p, name: p[name].data_ptr() if name in p else None                           # noqa: E731
        names = ("temperature", "top_k", "top_p", "min_p", "uniform")
        logits = _tensor(H, s["logits"], [case["vocab"], s["rows"]])
        draft = _tensor(H, s["draft_logits"], [case["vocab"], s["rows"]]) if case["drafter"] else None
        param = H.SampleParam(*(at(s["param"], n) for n in names))
        draft_param = H.SampleParam(*(at(s["draft_param"], n) for n in names)) if case["drafter"] else None
        need = L.spy_hip_sample_verify_scratch_size(C.byref(logits), case["seqs"])
        scratch = torch.empty(max(need, 1), dtype=torch.uint8, device="cuda")
        args = (None, C.byref(logits), C.byref(param), ref(draft), ref(draft_param), s["drafted"].data_ptr(), s["row_start"].data_ptr(), case["seqs"], s["accept"].data_ptr(),
                s["tokens"].data_ptr(), s["accepted"].data_ptr(), s["probs"].data_ptr(), scratch.data_ptr(), need)
        return {"call": L.spy_hip_sample_verify, "args": args, "keep": (logits, draft, param, draft_param, scratch), "check": H.check}
    nh, g, hd, ps, n_page = case["heads"], case["kv_heads"], case["hd"], case["page"], s["k_pages"].shape[0]
    batch = H.PagedBatch(case["seqs"], s["max_new"], s["max_kv"], s["row_start"].data_ptr(), s["kv_len"].data_ptr(), s["table"].data_ptr(), s["table"].shape[1])
    kp, vp = _tensor(H, s["k_pages"], [hd, ps, g, n_page]), _tensor(H, s["v_pages"], [ps, hd, g, n_page])
    ks = _tensor(H, s["k_scales"], [hd // 32, ps, g, n_page]) if "k_scales" in s else None
    vs = _tensor(H, s["v_scales"], [ps, hd // 32, g, n_page]) if "k_scales" in s else None
    q = _tensor(H, s["q"], [hd, nh, s["rows"]])
    if case["kind"] == "append":
        k, v, qo = _tensor(H, s["k"], [hd, g, s["rows"]]), _tensor(H, s["v"], [hd, g, s["rows"]]), _tensor(H, s["q_out"], [hd, nh, s["rows"]])
        rope = H.RopeParam(mode=case["mode"], num_dim=case["dims"], freq_base=case["base"], freq_scale=case["freq_scale"], attention_factor=1.0)
        args = tuple(C.byref(x) for x in (q, k, v, batch, rope, qo, kp, ks, vp, vs))
        return {"call": L.spy_hip_paged_append_q8, "args": (None,) + args, "keep": (q, k, v, batch, rope, qo, kp, ks, vp, vs), "check": H.check}
    out = _tensor(H, s["out"], [hd, nh, s["rows"]])
    tensors = (C.byref(q), C.byref(kp), ref(ks), C.byref(vp), ref(vs), C.byref(out), C.byref(batch))
    if case["kind"] == "shared":
        prefix = H.PagedPrefix(len(s["common"]), s["max_rows"], s["max_common"], s["seq_start"].data_ptr(), s["common"].data_ptr())
        need = L.spy_hip_paged_attention_shared_scratch_size(C.byref(q), C.byref(kp), C.byref(batch), C.byref(prefix))
        scratch = torch.empty(max(need, 1), dtype=torch.uint8, device="cuda")
        args = (None,) + tensors + (C.byref(prefix), 1.0 / math.sqrt(hd), scratch.data_ptr(), need)
        return {"call": L.spy_hip_paged_attention_shared, "args": args, "keep": (q, kp, ks, vp, vs, out, batch, prefix, scratch), "check": H.check}
    need = L.spy_hip_paged_attention_q8_scratch_size(C.byref(q), C.byref(kp), C.byref(batch))
    scratch = torch.empty(max(need, 1), dtype=torch.uint8, device="cuda")
    args = (None,) + tensors + (1.0 / math.sqrt(hd), 1, case["window"], scratch.data_ptr(), need)
    return {"call": L.spy_hip_paged_attention_q8, "args": args, "keep": (q, kp, ks, vp, vs, out, batch, scratch), "check": H.check}


def run(state):
    kind = state["case"]["kind"]
    if own:
        b = state.get("bound")
        if b is None:
            b = state["bound"] = _bind(state)
        b["check"](b["call"](*b["args"]))
        if kind == "verify":
            return {"tokens": state["tokens"], "accepted": state["accepted"], "probs": state["probs"]}
        return {"q": state["q_out"], **_read_back(state)} if kind == "append" else state["out"]
    return {"append": _append, "attend": _attend, "shared": _attend, "verify": _verify}[kind](state)


def work(case):
    if case["kind"] == "verify":
        rows, drafted = sum(_drafts(case)) + case["seqs"], sum(_drafts(case)) if case["drafter"] else 0
        return {"bytes": (rows + drafted) * 4 * case["vocab"] + rows * 44 + drafted * 16, "flops": 6 * (rows + drafted) * case["vocab"]}
    H, G, hd = case["heads"], case["kv_heads"], case["hd"]
    rows = sum(_lengths(case)[0])
    held = hd + hd // 16 if case.get("cache", "q8") == "q8" else 2 * hd                           # bytes of a K or V row in the cache
    if case["kind"] == "append":
        es = 4 if case["type"] == "f32" else 2
        return {"bytes": rows * (H * hd * (es + 2) + 2 * G * (hd * es + held)), "flops": rows * (3 * (H + G) * case["dims"] + 4 * G * hd)}
    pairs, read = _visible(case)
    return {"bytes": 2 * read * G * held + rows * H * hd * (2 + (4 if case["type"] == "f32" else 2)), "flops": 4 * pairs * H * hd}


# ---- from the definitions, in 64 bits -----------------------------------------------------------------------------------------------
def _exact_rotation(x, pos, case):
    """x: [heads][hd] of one token, as complex numbers turned by e^(i angle)"""
    nd = case["dims"]
    turn = np.exp(1j * pos * case["freq_scale"] * np.power(case["base"], -np.arange(0, nd, 2) / nd))
    y = x.copy()
    first, second = (slice(0, nd, 2), slice(1, nd, 2)) if case["mode"] == 0 else (slice(0, nd // 2), slice(nd // 2, nd))
    z = (x[:, first] + 1j * x[:, second]) * turn
    y[:, first], y[:, second] = z.real, z.imag
    return y


def _exact_blocks(x):
    """x: [heads][hd] as its blocks of 8 bits have it: the nearest multiples of d, d held as fp16"""
    b = x.reshape(x.shape[0], -1, 32)
    d = np.abs(b).max(axis=2, keepdims=True) / 127
    return (np.rint(b / np.where(d > 0, d, 1)) * d.astype(np.float16).astype(np.float64)).reshape(x.shape)


def _exact_values(q, d, axis):
    """pages on the host, in 64 bits; a value of the cache is held as fp16"""
    return (q.double().cpu().numpy() * np.repeat(d.double().cpu().numpy(), 32, axis=axis)).astype(np.float16).astype(np.float64)


def _exact_kept(x, param, r):
    """tokens of one row that its settings leave, and their probabilities"""
    get = lambda name, other: float(param[name][r]) if name in param else other                   # noqa: E731
    if get("temperature", 1.0) <= 0:
        return np.array([x.argmax()]), np.ones(1)
    by_rank = np.lexsort((np.arange(x.size), -x))
    k = int(get("top_k", 0))
    by_rank = by_rank[:k] if k > 0 else by_rank
    w = np.exp((x[by_rank] - x.max()) / get("temperature", 1.0))
    n, top_p = len(w), get("top_p", 1.0)
    if top_p < 1:
        n = int(np.searchsorted(np.cumsum(w), top_p * w.sum())) + 1
    n = max(1, min(n, int((w >= get("min_p", 0.0)).sum())))
    return by_rank[:n], w[:n] / w[:n].sum()


def _exact_verify(s):
    """the probabilities of the tokens that come out, request by request"""
    start, drafted = s["row_start"].cpu().numpy(), s["drafted"].cpu().numpy()
    probs, accept, uniform = np.zeros(s["rows"]), s["accept"].double().cpu().numpy(), s["param"]["uniform"].double().cpu().numpy()
    settings = [{n: x.double().cpu().numpy() for n, x in p.items()} for p in (s["param"], s["draft_param"])]
    for a, b in zip(start, start[1:]):
        for r in range(a, b):
            target, other = np.zeros(s["case"]["vocab"]), np.zeros(s["case"]["vocab"])
            at, p = _exact_kept(s["logits"][r].double().cpu().numpy(), settings[0], r)
            target[at] = p
            if r < b - 1:
                if "draft_logits" in s:
                    at, p = _exact_kept(s["draft_logits"][r].double().cpu().numpy(), settings[1], r)
                    other[at] = p
                else:
                    other[drafted[r]] = 1.0
                if accept[r] * other[drafted[r]] < target[drafted[r]]:
                    probs[r] = target[drafted[r]]
                    continue
            left = np.maximum(target - other, 0.0)
            upto = np.cumsum(left if left.any() else target)
            probs[r] = target[np.searchsorted(upto, uniform[r] * upto[-1], side="right")]
            break
    return {"tokens": None, "accepted": None, "probs": torch.tensor(probs)}


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "verify":
        return _exact_verify(s)
    news, kvs, _ = _lengths(case)
    ps, table, start = case["page"], s["table"].cpu().numpy(), np.concatenate([[0], np.cumsum(news)])
    if case["kind"] == "append":
        q, k, v = (s[n].double().cpu().numpy() for n in ("q", "k", "v"))
        kp, vp = _exact_values(s["k_pages"], s["k_scales"], 3), _exact_values(s["v_pages"], s["v_scales"], 2)
        for i, (new, kv) in enumerate(zip(news, kvs)):
            for t in range(new):
                row, pos = start[i] + t, kv - new + t
                page, at = table[i, pos // ps], pos % ps
                q[row] = _exact_rotation(q[row], pos, case)
                kp[page, :, at, :] = _exact_blocks(_exact_rotation(k[row], pos, case))
                vp[page, :, :, at] = _exact_blocks(v[row])
        return {"q": torch.tensor(q), "k_pages": torch.tensor(kp), "v_pages": torch.tensor(vp)}
    G, g, hd = case["kv_heads"], case["heads"] // case["kv_heads"], case["hd"]
    out = torch.zeros((s["rows"], case["heads"], hd), dtype=torch.float64, device="cuda")
    for i, (new, kv) in enumerate(zip(news, kvs)):
        pages = s["table"][i, :(kv + ps - 1) // ps].long()
        pos = torch.arange(kv - new, kv, device="cuda")[:, None]
        j = torch.arange(kv, device="cuda")[None]
        w = case.get("window", 0)
        hidden = (j > pos) | (j <= pos - w if w else j < 0)
        for h in range(G):
            k, v = s["k_pages"][pages, h].double(), s["v_pages"][pages, h].double()
            if "k_scales" in s:
                k = (k * s["k_scales"][pages, h].double().repeat_interleave(32, dim=2)).half().double()
                v = (v * s["v_scales"][pages, h].double().repeat_interleave(32, dim=1)).half().double()
            k, v = k.reshape(-1, hd)[:kv], v.transpose(1, 2).reshape(-1, hd)[:kv]
            x = torch.matmul(s["q"][start[i]:start[i] + new, h * g:(h + 1) * g].double().transpose(0, 1).reshape(-1, hd), k.t()) / math.sqrt(hd)
            x = x.masked_fill(hidden.repeat(g, 1), -math.inf)
            y = torch.exp(x - torch.logsumexp(x, dim=1, keepdim=True)) @ v
            out[start[i]:start[i] + new, h * g:(h + 1) * g] = y.reshape(g, new, hd).transpose(0, 1)
    return out
