"""The paged serving step, operator by operator: RoPE and the append of a chunk of new tokens into a paged KV
cache, attention of the chunk over that cache, and verification of drafted tokens against the target's
probabilities.

A batch is B sequences with their new tokens packed: rows q_start[b] .. q_start[b+1]-1 are sequence b's, its
token i at position len[b] + i.  The cache is a pool of pages, K and V each [n_pages][nkv][page][hd]; position t
of sequence b is slot t % page of page table[b][t // page].

run() computes the plain form in torch, or makes the framework's calls where `own` is true.  Sizes are those of
the two architectures in llamatov_amd/model.py (14 q / 2 KV heads of 64, vocabulary 151936; 32 / 8 of 128,
128256)."""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

F32, F64 = torch.float32, torch.float64
MAX_K = 1024          # candidates of a sampling distribution at most, as in lt_sample
THETA = {64: 1e6, 128: 5e5}


def listed():
    return [
        # one token of a short conversation on the small model: launch latency
        {"name": "attn-one-short", "kind": "attn", "B": 1, "n": 1, "ctx": 61, "nh": 14, "nkv": 2, "hd": 64, "page": 16,
         "kv": "f16", "window": 0, "ragged": False},
        # a draft of four tokens and the token before it, for each of eight conversations
        {"name": "attn-drafts-8", "kind": "attn", "B": 8, "n": 5, "ctx": 700, "nh": 32, "nkv": 8, "hd": 128, "page": 16,
         "kv": "f16", "window": 0, "ragged": False},
        # plain decode of a large batch, contexts of unequal lengths
        {"name": "attn-decode-64", "kind": "attn", "B": 64, "n": 1, "ctx": 4096, "nh": 32, "nkv": 8, "hd": 128,
         "page": 64, "kv": "f16", "window": 0, "ragged": False},
        # one token over a long document
        {"name": "attn-one-32k", "kind": "attn", "B": 1, "n": 1, "ctx": 32768, "nh": 32, "nkv": 8, "hd": 128, "page": 16,
         "kv": "f16", "window": 0, "ragged": False},
        # prompts in chunks of unequal lengths, contexts already cached
        {"name": "attn-chunks-4", "kind": "attn", "B": 4, "n": 509, "ctx": 6000, "nh": 32, "nkv": 8, "hd": 128,
         "page": 32, "kv": "f16", "window": 0, "ragged": True},
        # the last chunk of a 16k prompt: the largest product
        {"name": "attn-chunk-16k", "kind": "attn", "B": 1, "n": 2048, "ctx": 14336, "nh": 32, "nkv": 8, "hd": 128,
         "page": 64, "kv": "f16", "window": 0, "ragged": False},
        # an fp32 cache and a sliding window, on the small model
        {"name": "attn-f32-window", "kind": "attn", "B": 3, "n": 509, "ctx": 900, "nh": 14, "nkv": 2, "hd": 64,
         "page": 16, "kv": "f32", "window": 512, "ragged": True},
        # the append of one token, and of a batch of prompt chunks
        {"name": "append-one", "kind": "append", "B": 1, "n": 1, "ctx": 61, "nh": 14, "nkv": 2, "hd": 64, "page": 16,
         "kv": "f32", "ragged": False},
        {"name": "append-chunks", "kind": "append", "B": 4, "n": 700, "ctx": 2000, "nh": 32, "nkv": 8, "hd": 128,
         "page": 64, "kv": "f16", "ragged": True},
        # one conversation's four drafted tokens under the usual sampling settings
        {"name": "verify-one", "kind": "verify", "B": 1, "G": 4, "V": 151936, "T": 0.8, "top_k": 40, "top_p": 0.95,
         "drafter": True, "ragged": False},
        # a batch of conversations with a draft model
        {"name": "verify-64", "kind": "verify", "B": 64, "G": 4, "V": 151936, "T": 0.8, "top_k": 40, "top_p": 0.95,
         "drafter": True, "ragged": True},
        # drafts looked up in the text (no draft distribution), the widest candidate list
        {"name": "verify-lookup-16", "kind": "verify", "B": 16, "G": 7, "V": 128256, "T": 1.0, "top_k": 1024,
         "top_p": 1.0, "drafter": False, "ragged": True},
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["attn", "attn", "attn", "attn", "append", "verify", "verify"])
    if kind == "verify":
        B, G = _log_int(rng, 1, 64), rng.randrange(1, 8)
        V = rng.choice([151936, 128256, 4096, _log_int(rng, 500, 150000)])
        while B * (2 * G + 1) * V > 64 * 9 * 151936:
            B = max(1, B // 2)
        return {"kind": kind, "B": B, "G": G, "V": V, "T": rng.choice([0.0, 0.6, 0.8, 1.0, 1.3]),
                "top_k": rng.choice([1, 20, 40, 200, 1024]), "top_p": rng.choice([0.8, 0.95, 1.0]),
                "drafter": rng.random() < 0.6, "ragged": rng.random() < 0.6}
    nh, nkv, hd = rng.choice([(32, 8, 128), (32, 8, 128), (14, 2, 64)])
    c = {"kind": kind, "B": _log_int(rng, 1, 64), "nh": nh, "nkv": nkv, "hd": hd, "page": 1 << rng.randrange(3, 9),
         "kv": rng.choice(["f16", "f16", "f32"]), "ragged": rng.random() < 0.6}
    if kind == "append":
        return {**c, "n": _log_int(rng, 1, max(1, 4000 // c["B"])), "ctx": _log_int(rng, 1, 2000)}
    c["n"] = _log_int(rng, 1, max(1, 2048 // c["B"])) if rng.random() < 0.6 else rng.randrange(1, 9)
    c["ctx"] = _log_int(rng, 1, max(2, min(32768, 262144 // c["B"])))
    while c["B"] * c["n"] * (c["ctx"] + c["n"]) * nh * hd > 2048 * 14336 * 4096 // 2:
        c["ctx"] = max(1, c["ctx"] // 2)
    return {**c, "window": rng.choice([0, 0, 0, _log_int(rng, 1, 2048)])}


# ---- a batch's lengths -------------------------------------------------------------------------
def _spread(b):
    return 0.618034 * (b + 1) % 1


def _news(case):
    """New tokens of each sequence."""
    n, B = case["n"], case["B"]
    return [max(1, int(n * (0.25 + 0.75 * _spread(b + 3)))) if case["ragged"] else n for b in range(B)]


def _pasts(case):
    """Cached positions of each sequence before them: all of ctx for one, unequal for several."""
    B, ctx = case["B"], case["ctx"]
    return [ctx] if B == 1 else [max(0, int(ctx * (0.125 + 0.875 * _spread(b)))) for b in range(B)]


def _drafts(case):
    """Drafted tokens of each sequence."""
    return [(b * 3 + 1) % (case["G"] + 1) if case["ragged"] else case["G"] for b in range(case["B"])]


def _starts(news):
    return [sum(news[:b]) for b in range(len(news) + 1)]


# ---- inputs ------------------------------------------------------------------------------------
def _gen(seed, what):
    g = torch.Generator(device="cuda")
    g.manual_seed((int(seed) * 1000003 + what) & 0x7FFFFFFFFFFFFFFF)
    return g


def _normal(seed, what, *shape, std=1.0):
    return torch.randn(*shape, generator=_gen(seed, what), device="cuda") * std


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _cache(case, seed):
    """Pools that other requests' rows fill too, and a table of pages in no order."""
    B, nkv, hd, page = case["B"], case["nkv"], case["hd"], case["page"]
    news, pasts = _news(case), _pasts(case)
    need = [-(-(p + n) // page) for p, n in zip(pasts, news)]
    n_pages, cols = sum(need) + 3, max(need) + 1
    dt = torch.float16 if case["kv"] == "f16" else F32
    chan = 0.5 + 1.5 * torch.rand(nkv, 1, hd, generator=_gen(seed, 1), device="cuda")   # keys' channels differ in size
    k = (_normal(seed, 2, n_pages, nkv, page, hd) * chan).to(dt)
    v = _normal(seed, 3, n_pages, nkv, page, hd).to(dt)
    order = torch.randperm(n_pages, generator=_gen(seed, 4), device="cuda").tolist()
    table = np.full((B, cols), -1, np.int32)
    at = 0
    for b in range(B):
        table[b, :need[b]] = order[at:at + need[b]]
        at += need[b]
    return {"k": k, "v": v, "table": torch.from_numpy(table).cuda(), "q_start": _ints(_starts(news)),
            "len": _ints(pasts), "max_q": max(news), "max_len": max(p + n for p, n in zip(pasts, news))}


def prepare(case, seed):
    s = {"case": case, "kind": case["kind"]}
    if case["kind"] == "verify":
        return {**s, **_verify_inputs(case, seed)}
    s.update(_cache(case, seed))
    T, nh, nkv, hd = sum(_news(case)), case["nh"], case["nkv"], case["hd"]
    if case["kind"] == "attn":
        s["q"] = _normal(seed, 5, T, (nh + 2 * nkv) * hd)      # q|k|v rows of the projection, q rotated
        s["out"] = torch.empty(T, nh * hd, device="cuda")
    else:
        s["qkv"] = _normal(seed, 5, T, (nh + 2 * nkv) * hd)
        s["q_out"] = torch.empty(T, nh * hd, device="cuda")
        j = np.arange(hd // 2, dtype=np.float64)
        s["freqs"] = torch.from_numpy((THETA[hd] ** (-2.0 * j / hd)).astype(np.float32)).cuda()
    return s


def _verify_inputs(case, seed):
    B, V = case["B"], case["V"]
    rows = [d + 1 for d in _drafts(case)]
    T, start = sum(rows), _starts(rows)
    logits = _normal(seed, 1, T, V, std=2.5)
    hot = torch.randint(0, V, (T, 1), generator=_gen(seed, 2), device="cuda")           # a few likely tokens a row
    hot = (hot + torch.arange(12, device="cuda") * (V // 12)) % V
    logits.scatter_add_(1, hot, 6 + 4 * torch.rand(T, 12, generator=_gen(seed, 3), device="cuda"))
    near = torch.empty(T, V, device="cuda").normal_(generator=_gen(seed, 4)).mul_(0.6).add_(logits)   # the drafter's
    # a draft is drawn from the drafter's likely tokens (row r drafts token r + 1)
    top = near.topk(min(8, V), 1)
    pick = torch.multinomial(torch.softmax(top.values / 0.9, 1), 1, generator=_gen(seed, 5))
    drawn = top.indices.gather(1, pick)[:, 0].to(torch.int32)
    toks = torch.cat([drawn.new_zeros(1), drawn[:-1]])
    par = np.zeros(B, np.dtype([("temperature", "<f4"), ("top_k", "<i4"), ("top_p", "<f4"), ("reserved", "<i4"),
                                ("seed", "<u8"), ("counter", "<u8")]))
    par["temperature"], par["top_k"], par["top_p"] = case["T"], case["top_k"], case["top_p"]
    return {"logits": logits, "near": near if case["drafter"] else None, "toks": toks.contiguous(),
            "q_start": _ints(start), "max_q": max(rows), "params": torch.from_numpy(par.view(np.uint8).copy()).cuda(),
            "u": torch.rand(T, generator=_gen(seed, 6), device="cuda"),
            "out_tok": torch.empty(T, dtype=torch.int32, device="cuda"),
            "n_out": torch.empty(B, dtype=torch.int32, device="cuda")}


# ---- one pass ----------------------------------------------------------------------------------
def run(state):
    kind = state["kind"]
    if own:
        return {"attn": _own_attn, "append": _own_append, "verify": _own_verify}[kind](state)
    return {"attn": _plain_attn, "append": _plain_append, "verify": _plain_verify}[kind](state)


def _handles(s):
    """What a program on the framework keeps: its device tensors, the cache's descriptor, the workspace."""
    if "own" in s:
        return s["own"]
    from llamatov_amd import _lib, engine

    def dev(t, dtype):
        return None if t is None else engine.DevTensor(t.data_ptr(), t.shape, dtype, owns=False)

    c, h = s["case"], {"engine": engine}
    h["q_start"] = dev(s["q_start"], np.int32)
    B = c["B"]
    if s["kind"] == "verify":
        T, V = s["logits"].shape
        h.update(logits=dev(s["logits"], np.float32), near=dev(s["near"], np.float32), toks=dev(s["toks"], np.int32),
                 u=dev(s["u"], np.float32), params=dev(s["params"], np.uint8), out_tok=dev(s["out_tok"], np.int32),
                 n_out=dev(s["n_out"], np.int32))
        need = engine.verify_drafts_workspace_size(T, V, s["near"] is not None)
    else:
        kv_dtype, dt = (_lib.LT_KV_F16, np.uint16) if c["kv"] == "f16" else (_lib.LT_KV_F32, np.float32)
        h["len"] = dev(s["len"], np.int32)
        h["kv"] = engine.PagedKV(dev(s["k"], dt), dev(s["v"], dt), dev(s["table"], np.int32), kv_dtype)
        need = 0
        if s["kind"] == "attn":
            h.update(q=dev(s["q"], np.float32), out=dev(s["out"], np.float32))
            need = engine.attn_paged_workspace_size(s["q"].shape[0], B, c["nh"], h["kv"], s["max_q"], s["max_len"])
        else:
            h.update(qkv=dev(s["qkv"], np.float32), q_out=dev(s["q_out"], np.float32), freqs=dev(s["freqs"], np.float32))
    s["ws"] = torch.empty(max(need, 16), dtype=torch.uint8, device="cuda")
    h["ws"] = dev(s["ws"], np.uint8)
    torch.cuda.synchronize()
    s["own"] = h
    return h


def _own_attn(s):
    h, c = _handles(s), s["case"]
    h["engine"].attn_paged_into(h["q"], h["q_start"], h["len"], h["kv"], c["nh"], c["hd"] ** -0.5, h["out"],
                                max_q=s["max_q"], max_len=s["max_len"], window=c["window"], ws=h["ws"])
    return s["out"]


def _own_append(s):
    h, c = _handles(s), s["case"]
    h["engine"].rope_append_paged_into(h["qkv"], h["q_out"], h["q_start"], h["len"], c["nh"], h["freqs"], h["kv"])
    return [s["q_out"], s["k"], s["v"]]


def _own_verify(s):
    h = _handles(s)
    h["engine"].verify_drafts_into(h["logits"], h["toks"], h["q_start"], h["u"], h["params"], h["out_tok"], h["n_out"],
                                   draft_logits=h["near"], ws=h["ws"])
    return [s["out_tok"], s["n_out"]]


def _rows(s, T):
    """Sequence and number within it of each packed row."""
    r = torch.arange(T, device="cuda")
    b = torch.searchsorted(s["q_start"][1:].long(), r, right=True)
    return b, r - s["q_start"].long()[b]


def _plain_attn(s):
    c = s["case"]
    B, nh, nkv, hd, page, n = c["B"], c["nh"], c["nkv"], c["hd"], c["page"], s["max_q"]
    T, rep, L = s["q"].shape[0], nh // nkv, s["max_len"]
    pages = s["table"][:, :-(-L // page)].clamp(min=0).long()
    K = s["k"][pages].permute(0, 2, 1, 3, 4).reshape(B, nkv, -1, hd)[:, :, :L].to(F32)
    V = s["v"][pages].permute(0, 2, 1, 3, 4).reshape(B, nkv, -1, hd)[:, :, :L].to(F32)
    b, i = _rows(s, T)
    q = torch.zeros(B, n, nh, hd, device="cuda")
    q[b, i] = s["q"][:, :nh * hd].view(T, nh, hd)
    q = q.view(B, n, nkv, rep, hd).permute(0, 2, 3, 1, 4).reshape(B, nkv, rep * n, hd)
    S = torch.matmul(q, K.transpose(2, 3).contiguous()).mul_(hd ** -0.5).view(B, nkv, rep, n, L)
    p = s["len"].long()[:, None] + torch.arange(n, device="cuda")                      # [B][n]
    j = torch.arange(L, device="cuda")
    seen = j <= p[..., None]
    if c["window"]:
        seen &= j > p[..., None] - c["window"]
    S.masked_fill_(~seen[:, None, None], float("-inf"))
    S -= S.amax(-1, keepdim=True).clamp_(min=-1e30)
    S.exp_()
    z = S.sum(-1, keepdim=True)
    o = torch.matmul(S.view(B, nkv, rep * n, L), V).view(B, nkv, rep, n, hd) / z.clamp_(min=1e-30)
    o = o.permute(0, 3, 1, 2, 4).reshape(B, n, nh * hd)
    return o[b, i]


def _plain_append(s):
    c = s["case"]
    nh, nkv, hd, page = c["nh"], c["nkv"], c["hd"], c["page"]
    T = s["qkv"].shape[0]
    b, i = _rows(s, T)
    pos = s["len"].long()[b] + i
    # the framework's RoPE takes the angle as the binary32 product of the position and its frequency table (the cached
    # rows are then the same bits whichever path wrote them); its sine and cosine are taken in 64 bits
    a = (pos.to(F32)[:, None] * s["freqs"]).to(F64)
    cs, sn = a.cos().to(F32)[:, None], a.sin().to(F32)[:, None]
    x = s["qkv"].view(T, nh + 2 * nkv, hd)
    x1, x2 = x[:, :nh + nkv, :hd // 2], x[:, :nh + nkv, hd // 2:]
    r = torch.cat([x1 * cs - x2 * sn, x1 * sn + x2 * cs], -1)
    at = s["table"].long()[b, pos // page], slice(None), pos % page
    s["k"][at] = r[:, nh:].to(s["k"].dtype)
    s["v"][at] = x[:, nh + nkv:].to(s["v"].dtype)
    return [r[:, :nh].reshape(T, nh * hd), s["k"], s["v"]]


def _distribution(l, T, top_k, top_p):
    """Each row's candidates in rank order and their probabilities (0 past the nucleus)."""
    k = min(max(top_k, 1), MAX_K, l.shape[1]) if T > 0 else 1
    val, idx = torch.sort(l, dim=1, descending=True, stable=True)
    val, idx = val[:, :k], idx[:, :k]
    w = ((val.to(F64) - val[:, :1].to(F64)) / (np.float32(T).item() if T > 0 else 1.0)).exp_()
    cum = w.cumsum(1)
    if top_p < 1:
        before = torch.cat([torch.zeros_like(cum[:, :1]), cum[:, :-1]], 1)
        w = w.masked_fill(before >= np.float32(top_p).item() * cum[:, -1:], 0.0)
    return idx, w / w.sum(1, keepdim=True)


def _plain_verify(s):
    c = s["case"]
    T, B = s["logits"].shape[0], c["B"]
    start = s["q_start"].long()
    b, i = _rows(s, T)
    rows = start[1:] - start[:-1]
    ti, tp = _distribution(s["logits"], c["T"], c["top_k"], c["top_p"])
    nxt = torch.cat([s["toks"][1:], s["toks"][:1]]).long()                             # row r's draft
    if s["near"] is None:
        di, dp = nxt[:, None], torch.ones(T, 1, dtype=F64, device="cuda")
    else:
        di, dp = _distribution(s["near"], c["T"], c["top_k"], c["top_p"])
    p = torch.where(ti == nxt[:, None], tp, torch.zeros_like(tp)).sum(1)
    q = torch.where(di == nxt[:, None], dp, torch.zeros_like(dp)).sum(1)
    ok = (s["u"].to(F64) * q < p) & (i < rows[b] - 1)
    # accepted drafts of each sequence: those before its first row that is not ok
    first = torch.full((B,), T, dtype=torch.long, device="cuda").scatter_reduce_(
        0, b, torch.where(ok, torch.full_like(i, T), i), "amin")
    at = start[:-1] + first
    # the row the last token is drawn from: the target's less the drafter's, or the target's after the last draft
    P, I = tp[at], ti[at]
    dense = torch.zeros(B, c["V"], dtype=F64, device="cuda").scatter_(1, di[at], dp[at])
    R = (P - dense.gather(1, I)).clamp_(min=0)
    plain = (first == rows - 1) | (R.sum(1) <= 0)
    R = torch.where(plain[:, None], P, R)
    C = R.cumsum(1)
    u = s["u"].to(F64)[start[1:] - 1]
    last = I.gather(1, (C <= u[:, None] * C[:, -1:]).sum(1, keepdim=True).clamp_(max=I.shape[1] - 1))[:, 0]
    out = torch.where(i < first[b], nxt, torch.where(i == first[b], last[b], torch.full_like(nxt, -1)))
    return [out.to(torch.int32), (first + 1).to(torch.int32)]


# ---- what a pass cannot do without -------------------------------------------------------------
def work(case):
    if case["kind"] == "verify":
        d = _drafts(case)
        rows = sum(d) + case["B"] + (sum(d) if case["drafter"] else 0)
        return {"bytes": 4 * rows * case["V"], "flops": 2 * rows * case["V"]}
    nh, nkv, hd = case["nh"], case["nkv"], case["hd"]
    esz = 2 if case["kv"] == "f16" else 4
    news, pasts = _news(case), _pasts(case)
    T = sum(news)
    if case["kind"] == "append":
        return {"bytes": T * hd * (4 * (2 * nh + 2 * nkv) + 2 * nkv * esz), "flops": 3 * T * (nh + nkv) * hd}
    w = case["window"] or 1 << 40
    pairs = sum(sum(min(p + i + 1, w) for i in range(n)) for p, n in zip(pasts, news))
    cached = sum(p + n - max(0, p + 1 - w) for p, n in zip(pasts, news))
    return {"bytes": cached * 2 * nkv * hd * esz + 8 * T * nh * hd, "flops": 4 * nh * hd * pairs}


# ---- the definitions in 64 bits ----------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    start, pasts = s["q_start"].tolist(), None if case["kind"] == "verify" else s["len"].tolist()
    return {"attn": _exact_attn, "append": _exact_append, "verify": _exact_verify}[case["kind"]](case, s, start, pasts)


def _slots(s, b, n, page):
    t = torch.arange(n, device="cuda")
    return s["table"][b].long()[t // page], t % page


def _exact_attn(case, s, start, pasts):
    nh, nkv, hd = case["nh"], case["nkv"], case["hd"]
    out = torch.zeros(start[-1], nh, hd, dtype=F64, device="cuda")
    q = s["q"][:, :nh * hd].view(-1, nh, hd)
    for b in range(case["B"]):
        lo, hi = start[b], start[b + 1]
        end = pasts[b] + hi - lo
        pg, sl = _slots(s, b, end, case["page"])
        at = torch.arange(pasts[b], end, device="cuda")[:, None]
        key = torch.arange(end, device="cuda")[None]
        hidden = (key > at) | (key <= at - case["window"] if case["window"] else key < 0)
        for h in range(nh):
            K, V = s["k"][pg, h * nkv // nh, sl].to(F64), s["v"][pg, h * nkv // nh, sl].to(F64)
            x = (q[lo:hi, h].to(F64) @ K.t().contiguous() / math.sqrt(hd)).masked_fill(hidden, -math.inf)
            out[lo:hi, h] = torch.softmax(x, 1) @ V
    return out.view(-1, nh * hd)


def _exact_append(case, s, start, pasts):
    nh, nkv, hd, page = case["nh"], case["nkv"], case["hd"], case["page"]
    k, v = s["k"].to(F64), s["v"].to(F64)
    q_out = torch.empty(start[-1], nh * hd, dtype=F64, device="cuda")
    freqs = s["freqs"].cpu().numpy()
    for b in range(case["B"]):
        rows = s["qkv"][start[b]:start[b + 1]].to(F64).view(-1, nh + 2 * nkv, hd)
        at = np.arange(pasts[b], pasts[b] + len(rows))
        # by definition the angle is the binary32 product of the position and the table's frequency
        z = torch.from_numpy(np.exp(1j * (at.astype(np.float32)[:, None] * freqs).astype(np.float64))).cuda()[:, None]
        x = torch.complex(rows[:, :nh + nkv, :hd // 2].contiguous(), rows[:, :nh + nkv, hd // 2:].contiguous()) * z
        x = torch.cat([x.real, x.imag], -1)
        q_out[start[b]:start[b + 1]] = x[:, :nh].reshape(-1, nh * hd)
        pg, sl = _slots(s, b, pasts[b] + len(rows), page)
        pg, sl = pg[pasts[b]:], sl[pasts[b]:]
        k[pg, :, sl], v[pg, :, sl] = x[:, nh:], rows[:, nh + nkv:]
    return [q_out, k, v]


def _exact_verify(case, s, start, _):
    def ranked(l):
        """{token: probability} in rank order."""
        n = min(max(case["top_k"], 1), MAX_K, l.size) if case["T"] > 0 else 1
        cut = np.partition(l, l.size - n)[l.size - n]
        c = np.flatnonzero(l >= cut)
        c = c[np.lexsort((c, -l[c]))][:n]
        w = np.exp((l[c].astype(np.float64) - float(l[c[0]])) / (float(np.float32(case["T"])) or 1.0))
        total, run, m = w.sum(), 0.0, 0
        while m < n:
            run += w[m]
            m += 1
            if case["top_p"] < 1 and run >= float(np.float32(case["top_p"])) * total:
                break
        return dict(zip(c[:m].tolist(), (w[:m] / w[:m].sum()).tolist()))

    toks, u = s["toks"].tolist(), s["u"].double().tolist()
    out, n_out = [-1] * start[-1], []
    for b in range(case["B"]):
        r, end = start[b], start[b + 1] - 1
        while True:
            P = ranked(s["logits"][r].cpu().numpy())
            if r == end:
                Q = {}
                break
            x = toks[r + 1]
            Q = ranked(s["near"][r].cpu().numpy()) if case["drafter"] else {x: 1.0}
            if not u[r] * Q.get(x, 0.0) < P.get(x, 0.0):
                break
            out[r] = x
            r += 1
        R = {x: max(p - Q.get(x, 0.0), 0.0) for x, p in P.items()}
        R = R if sum(R.values()) > 0 else P
        goal, run = u[end] * math.fsum(R.values()), 0.0
        for x, p in R.items():
            run += p
            out[r] = x
            if run > goal:
                break
        n_out.append(r - start[b] + 1)
    return [torch.tensor(out, dtype=torch.int32), torch.tensor(n_out, dtype=torch.int32)]
