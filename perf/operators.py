"""Serving several requests at once, as cases that can be timed: new tokens rotated and appended to a paged cache, attention over
that cache for one or many new tokens of each request, and tokens drawn from the logits of a batch.

A case is a dict of plain values:
  kind      "append": spy_hip_paged_append, "attend": spy_hip_paged_attention, "sample": spy_hip_sample
  append, attend:
    seqs    requests in the batch; `chunks` of them bring up to `new` new tokens, the others one
    kv      the longest request's cached tokens, its new ones included; `ragged`: the others are shorter, else all alike
    heads, kv_heads, hd, page: query heads, K/V heads, their width, positions of a page
    type    append: type of q, k, v; attend: type of the output ("f32" or "f16"); mode: 0 neighbouring pairs, 2 halves; base, freq_scale, dims: the rotation
    window  attend: 0, or how many positions back a token sees
  sample:
    rows, vocab, filters ("all": temperature, top-k, top-p and min-p by row, some rows greedy, some with most tokens masked; "top_p": temperature and top-p)
"""
import ctypes as C
import math

import numpy as np
import torch

own = False


def listed():
    head = {"heads": 32, "kv_heads": 32, "hd": 128}
    group = {"heads": 32, "kv_heads": 8, "hd": 128}
    rope = {"base": 10000.0, "freq_scale": 1.0}
    return [
        # one request, one token: the smallest call there is
        {"name": "append_1", "kind": "append", "seqs": 1, "chunks": 0, "new": 1, "kv": 1001, "ragged": False, **head, "dims": 128, "page": 64, "type": "f32", "mode": 0, **rope},
        # a step of a full batch: a token for each of 64 requests, far into long sessions
        {"name": "append_64", "kind": "append", "seqs": 64, "chunks": 0, "new": 1, "kv": 8000, "ragged": True, **group, "dims": 128, "page": 16, "type": "f16", "mode": 2, **rope},
        # a prompt's chunk of the 7B shape
        {"name": "append_prompt_2048", "kind": "append", "seqs": 1, "chunks": 1, "new": 2048, "kv": 2048, "ragged": False, **head, "dims": 128, "page": 64, "type": "f32", "mode": 0, **rope},
        # the token loop's attention at the 7B shape: one request, 4096 cached tokens
        {"name": "attend_1_4096", "kind": "attend", "seqs": 1, "chunks": 0, "new": 1, "kv": 4096, "ragged": False, **head, "page": 64, "type": "f32", "window": 0},
        # a step of a full batch of requests of every length
        {"name": "attend_64_ragged", "kind": "attend", "seqs": 64, "chunks": 0, "new": 1, "kv": 4096, "ragged": True, **group, "page": 16, "type": "f16", "window": 0},
        # few requests with very long sessions, eight query heads to a K/V head
        {"name": "attend_8_30000", "kind": "attend", "seqs": 8, "chunks": 0, "new": 1, "kv": 30000, "ragged": True, "heads": 64, "kv_heads": 8, "hd": 128, "page": 128, "type": "f16", "window": 0},
        # a whole prompt of the 7B shape
        {"name": "attend_prompt_2048", "kind": "attend", "seqs": 1, "chunks": 1, "new": 2048, "kv": 2048, "ragged": False, **head, "page": 64, "type": "f16", "window": 0},
        # a chunk of a long document on what came before it
        {"name": "attend_512_on_7680", "kind": "attend", "seqs": 1, "chunks": 1, "new": 512, "kv": 8192, "ragged": False, **group, "page": 64, "type": "f16", "window": 0},
        # chunks of new requests between the single tokens of running ones, narrow heads, a window
        {"name": "attend_mixed", "kind": "attend", "seqs": 20, "chunks": 4, "new": 301, "kv": 1501, "ragged": True, "heads": 24, "kv_heads": 8, "hd": 64, "page": 32, "type": "f32", "window": 1024},
        # one row of the 7B vocabulary: what the token loop draws from
        {"name": "sample_1_32000", "kind": "sample", "rows": 1, "vocab": 32000, "filters": "all"},
        # a batch of requests with settings of their own
        {"name": "sample_64_32000", "kind": "sample", "rows": 64, "vocab": 32000, "filters": "all"},
        # a large batch over a large vocabulary of odd size, nothing cut by rank
        {"name": "sample_256_100003", "kind": "sample", "rows": 256, "vocab": 100003, "filters": "top_p"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["append", "attend", "attend", "sample"])
    if kind == "sample":
        vocab = _log(rng, 1000, 131072)
        return {"kind": kind, "rows": min(_log(rng, 1, 256), 256 * 100003 // vocab), "vocab": vocab, "filters": rng.choice(["all", "top_p"])}
    heads, kv_heads = rng.choice([(32, 32), (32, 8), (24, 8), (16, 1), (10, 2), (8, 8)])
    shape = {"heads": heads, "kv_heads": kv_heads, "hd": rng.choice([64, 128, 128, 256]), "page": rng.choice([16, 32, 64, 128, 256])}
    if kind == "append":
        new = rng.choice([1, _log(rng, 2, 700)])
        seqs = _log(rng, 1, 64) if new == 1 else min(_log(rng, 1, 8), max(1, 1500 // new))
        return {"kind": kind, "seqs": seqs, "chunks": 0 if new == 1 else rng.randint(1, seqs), "new": new, "kv": new + _log(rng, 1, 20000), "ragged": rng.random() < 0.5, **shape,
                "dims": shape["hd"] // rng.choice([1, 1, 2]), "type": rng.choice(["f32", "f16"]), "mode": rng.choice([0, 2]), "base": rng.choice([10000.0, 500000.0]),
                "freq_scale": rng.choice([1.0, 0.25])}
    shape["hd"] = min(shape["hd"], 128) if kv_heads == 32 else shape["hd"]
    wide = kv_heads * shape["hd"] / 1024
    if rng.random() < 0.5:
        seqs, new, chunks = _log(rng, 1, 64), 1, 0
    else:
        seqs, new = _log(rng, 1, 16), _log(rng, 2, 1000)
        chunks = rng.randint(1, seqs)
    most = int(min(30000, 150000 / wide / seqs, 1.5e10 / (seqs * heads * new * shape["hd"])))
    if most <= new:
        seqs = chunks = 1
        most = int(min(30000, 150000 / wide, 1.5e10 / (heads * new * shape["hd"])))
    kv = max(new, _log(rng, 16, max(17, most)))
    return {"kind": kind, "seqs": seqs, "chunks": chunks, "new": new, "kv": kv, "ragged": rng.random() < 0.7, **shape, "type": rng.choice(["f16", "f16", "f32"]),
            "window": rng.choice([0, 0, _log(rng, 16, 4096)])}


def _lengths(case):
    """(new tokens, cached tokens) of each request, from the case alone: every length between a fifth of the longest and the longest, the first one the longest"""
    news, kvs = [], []
    for i in range(case["seqs"]):
        part = 1.0 - 0.8 * ((i * 0.6180339887) % 1.0) if case["ragged"] else 1.0
        new = max(1, int(case["new"] * part)) if i < case["chunks"] else 1
        news.append(new)
        kvs.append(max(new, int(case["kv"] * part)))
    return news, kvs


def _visible(case):
    """pairs of a query token and a cached token that it sees, and the cached tokens that any token of a request sees"""
    pairs = read = 0
    for new, kv in zip(*_lengths(case)):
        w = case["window"] or kv
        pairs += sum(min(p + 1, w) for p in range(kv - new, kv))
        read += min(kv, w + new - 1)
    return pairs, read


def _params(case, gen):
    rows = case["rows"]

    def pick(values):
        return torch.tensor(values, device="cuda")[torch.randint(0, len(values), (rows,), generator=gen, device="cuda")]

    p = {"temperature": torch.rand(rows, generator=gen, device="cuda") + 0.5, "top_p": pick([0.5, 0.9, 0.95]), "uniform": torch.rand(rows, generator=gen, device="cuda")}
    if case["filters"] == "all":
        p["top_k"] = pick([20, 40, 50, 500, 0]).to(torch.int32)
        p["min_p"] = pick([0.0, 0.05, 0.1])
        p["top_p"] = torch.where(torch.rand(rows, generator=gen, device="cuda") < 0.3, torch.ones_like(p["top_p"]), p["top_p"])
        p["temperature"][9::16] = 0.0
    return p


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    randn = lambda *shape: torch.randn(shape, generator=gen, device="cuda")                     # noqa: E731
    s = {"case": case}
    if case["kind"] == "sample":
        rows, vocab = case["rows"], case["vocab"]
        s["logits"] = randn(rows, vocab) * 2.5
        at = torch.randint(0, vocab, (rows, 24), generator=gen, device="cuda")                   # the tokens that a context makes likely
        s["logits"].scatter_add_(1, at, 4.0 + 5.0 * torch.rand((rows, 24), generator=gen, device="cuda"))
        if case["filters"] == "all" and rows > 5:                                                 # a grammar leaves a few tokens
            s["logits"][5::8].masked_fill_(torch.rand((len(range(5, rows, 8)), vocab), generator=gen, device="cuda") > 60 / vocab, -math.inf)
            s["logits"][5::8, 7] = 1.0
        s.update(_params(case, gen))
        s["token"] = torch.zeros(rows, dtype=torch.int32, device="cuda")
        s["prob"] = torch.zeros(rows, device="cuda")
        return s
    news, kvs = _lengths(case)
    H, G, hd, ps, rows = case["heads"], case["kv_heads"], case["hd"], case["page"], sum(news)
    append = case["kind"] == "append"
    first = [(kv - new) // ps if append else 0 for new, kv in zip(news, kvs)]                     # pages that the call does not touch are not kept here
    count = [(kv + ps - 1) // ps - f for kv, f in zip(kvs, first)]
    n_page, width = sum(count) + 3, max((kv + ps - 1) // ps for kv in kvs)
    order = np.random.default_rng(seed).permutation(n_page)
    table, at = np.zeros((len(kvs), width), np.int32), 0
    for i, (f, c) in enumerate(zip(first, count)):
        table[i, f:f + c] = order[at:at + c]
        at += c
    i32 = lambda v: torch.tensor(np.asarray(v, np.int32), device="cuda")                         # noqa: E731
    s.update(row_start=i32(np.concatenate([[0], np.cumsum(news)])), kv_len=i32(kvs), table=i32(table), rows=rows, max_new=max(news), max_kv=max(kvs))
    s["k_pages"] = torch.empty((n_page, G, ps, hd), dtype=torch.float16, device="cuda").normal_(generator=gen)
    s["v_pages"] = torch.empty((n_page, G, hd, ps), dtype=torch.float16, device="cuda").normal_(generator=gen)
    if append:
        dt = torch.float32 if case["type"] == "f32" else torch.float16
        s["q"], s["k"], s["v"] = randn(rows, H, hd).to(dt), randn(rows, G, hd).to(dt), randn(rows, G, hd).to(dt)
        s["q_out"] = torch.zeros((rows, H, hd), dtype=torch.float16, device="cuda")
    else:
        s["q"] = (randn(rows, H, hd) * 1.5).half()
        s["out"] = torch.zeros((rows, H, hd), dtype=torch.float32 if case["type"] == "f32" else torch.float16, device="cuda")
    return s


# ---- the plain forms ----------------------------------------------------------------------------------------------------------------
def _positions(s):
    """request and position of every new token"""
    row = torch.arange(s["rows"], device="cuda")
    seq = torch.searchsorted(s["row_start"][1:].long(), row, right=True)
    end = s["row_start"].long()[seq + 1]
    return seq, s["kv_len"].long()[seq] - (end - row)


def _rotated(x, pos, case):
    nd = case["dims"]
    i = torch.arange(nd // 2, device="cuda", dtype=torch.float64)
    angle = pos.double()[:, None] * (case["freq_scale"] * case["base"] ** (-2.0 * i / nd))        # far positions: 64 bits
    c, s = torch.cos(angle).float()[:, None, :], torch.sin(angle).float()[:, None, :]
    x = x.float()
    a, b = (x[..., 0:nd:2], x[..., 1:nd:2]) if case["mode"] == 0 else (x[..., :nd // 2], x[..., nd // 2:nd])
    u, v = a * c - b * s, a * s + b * c
    y = torch.stack([u, v], dim=-1).flatten(-2) if case["mode"] == 0 else torch.cat([u, v], dim=-1)
    return torch.cat([y, x[..., nd:]], dim=-1).half()


def _append(s):
    case, ps = s["case"], s["case"]["page"]
    seq, pos = _positions(s)
    page, at = s["table"][seq, pos // ps].long(), pos % ps
    s["k_pages"][page, :, at, :] = _rotated(s["k"], pos, case)
    s["v_pages"][page, :, :, at] = s["v"].half()
    return {"q": _rotated(s["q"], pos, case), "k_pages": s["k_pages"], "v_pages": s["v_pages"]}


def _attend(s):
    case, ps = s["case"], s["case"]["page"]
    H, G, hd, n = case["heads"], case["kv_heads"], case["hd"], case["seqs"]
    j = torch.arange(s["max_kv"], device="cuda")
    page, at = s["table"][:, j // ps].long(), (j % ps).expand(n, -1)
    k = s["k_pages"][page, :, at, :].permute(0, 2, 1, 3).float()                                  # [request][K/V head][position][hd]
    v = s["v_pages"][page, :, :, at].permute(0, 2, 1, 3).float()
    start, kv = s["row_start"].long(), s["kv_len"].long()
    i = torch.arange(s["max_new"], device="cuda")
    there = i[None, :] < (start[1:] - start[:-1])[:, None]
    row = (start[:-1, None] + i).clamp(max=s["rows"] - 1)
    q = s["q"][row].float().reshape(n, -1, G, H // G, hd).permute(0, 2, 1, 3, 4).reshape(n, G, -1, hd)
    pos = (kv - (start[1:] - start[:-1]))[:, None] + i                                            # [request][new token]
    seen = (j <= pos[..., None]) & (j < kv[:, None, None])
    if case["window"]:
        seen &= j > pos[..., None] - case["window"]
    seen = seen.repeat_interleave(H // G, dim=1)[:, None]                                         # [request][1][token, head of the group][position]
    x = torch.matmul(q, k.transpose(2, 3)).mul_(1.0 / math.sqrt(hd)).masked_fill_(~seen, -math.inf)
    top = x.amax(dim=-1, keepdim=True)
    e = x.sub_(torch.where(top > -math.inf, top, torch.zeros_like(top))).exp_()
    total = e.sum(dim=-1, keepdim=True)
    o = torch.matmul(e, v) / torch.where(total > 0, total, torch.ones_like(total))
    o = o.reshape(n, G, -1, H // G, hd).permute(0, 2, 1, 3, 4).reshape(n, -1, H, hd)
    return o[there].to(s["out"].dtype)


def _sample(s):
    x = s["logits"].double()                                                                      # sums next to a border: 64 bits
    rows, vocab = x.shape
    y, order = torch.sort(x, dim=1, descending=True, stable=True)
    t = s["temperature"].double()[:, None]
    greedy = t <= 0
    w = torch.exp((y - y[:, :1]) / torch.where(greedy, torch.ones_like(t), t))
    rank = torch.arange(vocab, device="cuda")[None]
    if "top_k" in s:
        k = s["top_k"].long()[:, None]
        w = torch.where((k > 0) & (rank >= k), torch.zeros_like(w), w)
    before = torch.cumsum(w, dim=1) - w
    p = s["top_p"].double()[:, None]
    keep = (p >= 1) | (before < p * w.sum(dim=1, keepdim=True))
    if "min_p" in s:
        keep &= w >= s["min_p"].double()[:, None]
    keep = torch.where(greedy, rank == 0, keep | (rank == 0))
    w = torch.zeros_like(w).scatter_(1, order, torch.where(keep, w, torch.zeros_like(w)))         # back in the vocabulary's order
    run_ = torch.cumsum(w, dim=1)
    total = run_[:, -1:]
    token = (run_ > s["uniform"].double()[:, None] * total).to(torch.uint8).argmax(dim=1)
    return {"token": token.to(torch.int32), "prob": (w.gather(1, token[:, None]) / total)[:, 0].float()}


# ---- the framework's calls ----------------------------------------------------------------------------------------------------------
def _tensor(H, x, dims):
    t = {torch.float32: H.F32, torch.float16: H.F16}[x.dtype]
    return H.tensor(x.data_ptr(), t, dims)


def _bind(s):
    """What a program that serves requests keeps beside its buffers: their descriptions and the workspace."""
    from spy_amd import _lib as H
    H.init(0)
    L, case = H.load(), s["case"]
    if case["kind"] == "sample":
        logits = _tensor(H, s["logits"], [case["vocab"], case["rows"]])
        at = lambda name: s[name].data_ptr() if name in s else None                              # noqa: E731
        param = H.SampleParam(at("temperature"), at("top_k"), at("top_p"), at("min_p"), at("uniform"))
        need = L.spy_hip_sample_scratch_size(C.byref(logits))
        scratch = torch.empty(max(need, 1), dtype=torch.uint8, device="cuda")
        args = (None, C.byref(logits), C.byref(param), s["token"].data_ptr(), s["prob"].data_ptr(), scratch.data_ptr(), need)
        return {"call": L.spy_hip_sample, "args": args, "out": {"token": s["token"], "prob": s["prob"]}, "keep": (logits, param, scratch), "check": H.check}
    nh, g, hd, ps, n_page = case["heads"], case["kv_heads"], case["hd"], case["page"], s["k_pages"].shape[0]
    batch = H.PagedBatch(case["seqs"], s["max_new"], s["max_kv"], s["row_start"].data_ptr(), s["kv_len"].data_ptr(), s["table"].data_ptr(), s["table"].shape[1])
    kp, vp = _tensor(H, s["k_pages"], [hd, ps, g, n_page]), _tensor(H, s["v_pages"], [ps, hd, g, n_page])
    q = _tensor(H, s["q"], [hd, nh, s["rows"]])
    if case["kind"] == "append":
        k, v, qo = _tensor(H, s["k"], [hd, g, s["rows"]]), _tensor(H, s["v"], [hd, g, s["rows"]]), _tensor(H, s["q_out"], [hd, nh, s["rows"]])
        rope = H.RopeParam(mode=case["mode"], num_dim=case["dims"], freq_base=case["base"], freq_scale=case["freq_scale"], attention_factor=1.0)
        args = tuple(C.byref(x) for x in (q, k, v, batch, rope, qo, kp, vp))
        return {"call": L.spy_hip_paged_append, "args": (None,) + args, "out": {"q": s["q_out"], "k_pages": s["k_pages"], "v_pages": s["v_pages"]},
                "keep": (q, k, v, batch, rope, qo, kp, vp), "check": H.check}
    out = _tensor(H, s["out"], [hd, nh, s["rows"]])
    need = L.spy_hip_paged_attention_scratch_size(C.byref(q), C.byref(kp), C.byref(batch))
    scratch = torch.empty(max(need, 1), dtype=torch.uint8, device="cuda")
    args = (None, C.byref(q), C.byref(kp), C.byref(vp), C.byref(out), C.byref(batch), 1.0 / math.sqrt(hd), 1, case["window"], scratch.data_ptr(), need)
    return {"call": L.spy_hip_paged_attention, "args": args, "out": s["out"], "keep": (q, kp, vp, out, batch, scratch), "check": H.check}


def run(state):
    if own:
        b = state.get("bound")
        if b is None:
            b = state["bound"] = _bind(state)
        b["check"](b["call"](*b["args"]))
        return b["out"]
    return {"append": _append, "attend": _attend, "sample": _sample}[state["case"]["kind"]](state)


def work(case):
    if case["kind"] == "sample":
        return {"bytes": case["rows"] * (4 * case["vocab"] + 28), "flops": 6 * case["rows"] * case["vocab"]}
    H, G, hd = case["heads"], case["kv_heads"], case["hd"]
    rows = sum(_lengths(case)[0])
    if case["kind"] == "append":
        return {"bytes": rows * (H + 2 * G) * hd * ((4 if case["type"] == "f32" else 2) + 2), "flops": 3 * rows * (H + G) * case["dims"]}
    pairs, read = _visible(case)
    return {"bytes": 4 * read * G * hd + rows * H * hd * (2 + (4 if case["type"] == "f32" else 2)), "flops": 4 * pairs * H * hd}


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


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "sample":
        prob = np.zeros(case["rows"])
        for r in range(case["rows"]):
            x = s["logits"][r].double().cpu().numpy()
            get = lambda name, other: float(s[name][r]) if name in s else other                  # noqa: E731
            t, u = get("temperature", 1.0), get("uniform", 0.0)
            if t <= 0:
                prob[r] = 1.0
                continue
            by_rank = np.lexsort((np.arange(x.size), -x))
            k = int(get("top_k", 0))
            by_rank = by_rank[:k] if k > 0 else by_rank
            w = np.exp((x[by_rank] - x.max()) / t)
            n, top_p = len(w), get("top_p", 1.0)
            if top_p < 1:
                n = int(np.searchsorted(np.cumsum(w), top_p * w.sum())) + 1
            n = max(1, min(n, int((w >= get("min_p", 0.0)).sum())))
            kept = np.sort(by_rank[:n])
            w = np.exp((x[kept] - x.max()) / t)
            at = int(np.searchsorted(np.cumsum(w), u * w.sum(), side="right"))
            prob[r] = w[min(at, n - 1)] / w.sum()
        return {"token": None, "prob": torch.tensor(prob)}
    news, kvs = _lengths(case)
    ps, table, start = case["page"], s["table"].cpu().numpy(), np.concatenate([[0], np.cumsum(news)])
    if case["kind"] == "append":
        q, k, v = (s[n].double().cpu().numpy() for n in ("q", "k", "v"))
        kp, vp = s["k_pages"].double().cpu().numpy(), s["v_pages"].double().cpu().numpy()
        for i, (new, kv) in enumerate(zip(news, kvs)):
            for t in range(new):
                row, pos = start[i] + t, kv - new + t
                page, at = table[i, pos // ps], pos % ps
                q[row] = _exact_rotation(q[row], pos, case)
                kp[page, :, at, :] = _exact_rotation(k[row], pos, case)
                vp[page, :, :, at] = v[row]
        return {"q": torch.tensor(q), "k_pages": torch.tensor(kp), "v_pages": torch.tensor(vp)}
    G, g, hd = case["kv_heads"], case["heads"] // case["kv_heads"], case["hd"]
    out = torch.zeros((s["rows"], case["heads"], hd), dtype=torch.float64, device="cuda")
    for i, (new, kv) in enumerate(zip(news, kvs)):
        pages = s["table"][i, :(kv + ps - 1) // ps].long()
        pos = torch.arange(kv - new, kv, device="cuda")[:, None]
        j = torch.arange(kv, device="cuda")[None]
        hidden = (j > pos) | (j <= pos - case["window"] if case["window"] else j < 0)
        for h in range(G):
            k = s["k_pages"][pages, h].reshape(-1, hd)[:kv].double()
            v = s["v_pages"][pages, h].transpose(1, 2).reshape(-1, hd)[:kv].double()
            for c in range(h * g, (h + 1) * g):
                x = (s["q"][start[i]:start[i] + new, c].double() @ k.t()) / math.sqrt(hd)
                x = x.masked_fill(hidden, -math.inf)
                out[start[i]:start[i] + new, c] = torch.exp(x - torch.logsumexp(x, dim=1, keepdim=True)) @ v
    return out
