"""Verification of drafts (lt_verify.hip) against a plain float64 statement of its rule: every token and count, over
vocabulary sizes on both sides of the slices, ragged batches, tied and non-finite logits, greedy and nucleus settings,
drafts with and without a distribution, the generator's numbers, and the frequencies of the drawn tokens."""
import ctypes

import numpy as np
import pytest

from llamatov_amd import _lib
from llamatov_amd import engine as dr
from llamatov_amd._lib import call

pytestmark = pytest.mark.gpu

PARAM_DT = np.dtype([("temperature", "<f4"), ("top_k", "<i4"), ("top_p", "<f4"), ("reserved", "<i4"),
                     ("seed", "<u8"), ("counter", "<u8")])


def case(msg):
    print(f"[gpu-case] {msg}", flush=True)


def ranked(l, T, top_k, top_p):
    """(candidates in rank order, their probabilities)."""
    T, top_p = float(np.float32(T)), float(np.float32(top_p))
    l = l + np.float32(0)                                   # -0 and +0 tie
    with np.errstate(all="ignore"):
        inv = np.float32(1) / np.float32(T) if T > 0 else np.float32(np.inf)
    k = min(max(top_k, 1), 1024, l.size) if T > 0 and np.isfinite(inv) else 1
    order = np.argsort(-l, kind="stable")[:k]
    if not np.isfinite(l[order[0]]):
        k, order = 1, order[:1]
    w = np.ones(1) if k == 1 else np.exp((l[order].astype(np.float64) - float(l[order[0]])) / T)
    c = np.cumsum(w)
    n = k if top_p >= 1 else int(np.argmax(c >= top_p * c[-1])) + 1
    return order[:n], w[:n] / c[n - 1]


def philox(counter, seed):
    c = [counter & 0xFFFFFFFF, counter >> 32, 0, 0]
    k = [seed & 0xFFFFFFFF, seed >> 32]
    for r in range(10):
        if r:
            k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
        p0, p1 = 0xD2511F53 * c[0], 0xCD9E8D57 * c[2]
        c = [(p1 >> 32) ^ c[1] ^ k[0], p1 & 0xFFFFFFFF, (p0 >> 32) ^ c[3] ^ k[1], p0 & 0xFFFFFFFF]
    return (c[0] >> 8) * 2.0 ** -24


def verify(logits, dlogits, toks, start, u, params):
    out, n_out = np.full(len(toks), -1, np.int32), []
    for b in range(len(start) - 1):
        r, end = start[b], start[b + 1] - 1
        if end < r:
            n_out.append(0)
            continue
        P = params[b]
        args = (P["temperature"], int(P["top_k"]), P["top_p"])
        while True:
            ids, p = ranked(logits[r], *args)
            if r == end:
                w = p
                break
            x = toks[r + 1]
            if dlogits is None:
                q = {int(x): 1.0}
            else:
                q = dict(zip(*(v.tolist() for v in ranked(dlogits[r], *args))))
            px = dict(zip(ids.tolist(), p.tolist())).get(int(x), 0.0)
            if not float(u[r]) * q.get(int(x), 0.0) < px:
                w = np.maximum(p - np.array([q.get(int(i), 0.0) for i in ids]), 0)
                break
            out[r] = x
            r += 1
        if not w.sum() > 0:
            w = p
        c = np.cumsum(w)
        hit = np.flatnonzero(c > float(u[end]) * c[-1])
        out[r] = ids[hit[0] if len(hit) else -1]
        n_out.append(r - start[b] + 1)
    return out, np.asarray(n_out, np.int32)


def run(gpu, logits, dlogits, toks, start, u, params, lens=None):
    T, V = logits.shape
    B = len(start) - 1
    D = dr.DevTensor.from_host
    n = dr.verify_drafts_workspace_size(T, V, dlogits is not None)
    ws = D(np.full(max(n, 8), 0xA5, np.uint8), gpu)
    t = {"l": D(logits, gpu), "d": None if dlogits is None else D(dlogits, gpu), "t": D(toks, gpu), "s": D(start, gpu),
         "u": None if u is None else D(u, gpu), "p": D(params.view(np.uint8), gpu),
         "o": D(np.full(T, -9, np.int32), gpu), "n": D(np.full(B, -9, np.int32), gpu),
         "len": None if lens is None else D(lens, gpu)}
    dr.verify_drafts_into(t["l"], t["t"], t["s"], t["u"], t["p"], t["o"], t["n"], ws, draft_logits=t["d"], lens=t["len"])
    got = t["o"].to_host(), t["n"].to_host(), t["p"].to_host().view(PARAM_DT), None if lens is None else t["len"].to_host()
    ws.free()
    for v in t.values():
        if v is not None:
            v.free()
    return got


def batch(rng, V, rows, settings, drafter, ties=False, near=0.6):
    """Logits with a few likely tokens a row, a drafter near them, drafts drawn from its distribution."""
    T, start = sum(rows), np.cumsum([0] + list(rows)).astype(np.int32)
    logits = (rng.standard_normal((T, V)) * 2.5).astype(np.float32)
    for r in range(T):
        logits[r, rng.integers(0, V, 8)] += 7
    if ties:
        logits = np.round(logits)
    dl = (logits + near * rng.standard_normal((T, V))).astype(np.float32)
    if ties:
        dl = np.round(dl)
    params = np.zeros(len(rows), PARAM_DT)
    toks = np.zeros(T, np.int32)
    for b in range(len(rows)):
        s = settings[b % len(settings)]
        params[b]["temperature"], params[b]["top_k"], params[b]["top_p"] = s
        params[b]["seed"], params[b]["counter"] = 77 + b, (b << 33) + 5
        for r in range(start[b], start[b + 1] - 1):
            ids, p = ranked(dl[r], s[0], s[1], s[2])
            toks[r + 1] = rng.choice(ids, p=p)
    return logits, dl if drafter else None, toks, start, rng.random(T).astype(np.float32), params


SETTINGS = [(0.8, 40, 0.95), (0.0, 40, 1.0), (1.0, 1024, 1.0), (1.3, 300, 0.8), (0.7, 1, 1.0), (1.0, 5000, 0.999),
            (1e-39, 40, 0.9), (0.9, 17, 1e-7)]


@pytest.mark.parametrize("drafter", [True, False])
@pytest.mark.parametrize("V", [1, 2, 60, 1000, 8192, 8193, 40000, 151936])
def test_verification_matches(gpu, V, drafter):
    rng = np.random.default_rng(V)
    for ties in (False, True):
        rows = [5, 1, 0, 3, 2, 8, 4, 1, 2, 6]
        case(f"verify V={V} drafter={drafter} ties={ties}")
        b = batch(rng, V, rows, SETTINGS, drafter, ties)
        lens = np.arange(10, 20).astype(np.int32)
        out, n, par, ln = run(gpu, *b, lens=lens)
        eo, en = verify(*b)
        assert np.array_equal(n, en), (n, en)
        assert np.array_equal(out, eo), np.flatnonzero(out != eo)
        assert np.array_equal(ln, lens + en)
        assert np.array_equal(par, b[-1])                   # given numbers: the counters stay


@pytest.mark.parametrize("V", [3000, 32768, 128256])
def test_verification_large_batch(gpu, V):
    """Enough rows for the wide slices; many equal rows of a drafter that agrees."""
    case(f"verify 70 sequences V={V}")
    rng = np.random.default_rng(V + 1)
    rows = [int(v) for v in rng.integers(0, 7, 70)]
    if V == 128256:
        rows = rows[:24]
    b = batch(rng, V, rows, SETTINGS, True, near=0.3)
    out, n, _, _ = run(gpu, *b)
    eo, en = verify(*b)
    assert np.array_equal(n, en) and np.array_equal(out, eo)


@pytest.mark.parametrize("V", [4100, 16384, 16387, 65540, 131072, 200001])
def test_verification_runs_of_large_neighbours(gpu, V):
    """Logits in ascending, descending and equal order, and blocks of equal large ones: far more of them at or above the
    bound of the groups than are candidates."""
    case(f"verify runs V={V}")
    rng = np.random.default_rng(V)
    settings = [(1.0, 1024, 1.0), (0.7, 40, 0.9), (1.0, 1000, 0.99)]
    b = batch(rng, V, [3, 3, 3, 3, 2], settings, True)
    for l in (b[0], b[1]):
        up = (np.arange(V) * np.float32(2e-4)).astype(np.float32)
        l[0:3] = up
        l[3:6] = up[::-1]
        l[6:9] = 1.5
        l[9:12, V // 3:V // 3 + 3000] = 9.0
        l[9, V - 1] = 9.5
        l[12:, :4000] = np.floor(up[:4000] * 50)
    toks = b[2]
    toks[1], toks[4], toks[7], toks[10], toks[13] = V - 3, 2, 5, V // 3 + 7, 3999
    out, n, _, _ = run(gpu, *b)
    eo, en = verify(*b)
    assert np.array_equal(n, en) and np.array_equal(out, eo)


def test_verification_agreeing_drafter_accepts_all(gpu):
    case("verify equal logits")
    rng = np.random.default_rng(5)
    b = list(batch(rng, 5000, [6] * 12, SETTINGS, True, near=0.0))
    b[4] = np.full(len(b[2]), 1 - 2.0 ** -24, np.float32)    # the largest u there is
    out, n, _, _ = run(gpu, *b)
    assert np.all(n == 6)
    for s in range(12):
        assert np.array_equal(out[6 * s:6 * s + 5], b[2][6 * s + 1:6 * s + 6])


def test_verification_generator(gpu):
    """Numbers from each sequence's state: Philox at counter + row, the counter advanced by the rows."""
    case("verify philox")
    rng = np.random.default_rng(6)
    rows = [5, 1, 0, 3, 2, 8]
    b = list(batch(rng, 2000, rows, SETTINGS, True))
    b[4] = None
    out, n, par, _ = run(gpu, *b)
    u = np.concatenate([[philox(int(p["counter"]) + i, int(p["seed"])) for i in range(m)] for p, m in zip(b[5], rows)])
    b[4] = u
    eo, en = verify(*b)
    assert np.array_equal(n, en) and np.array_equal(out, eo)
    assert np.array_equal(par["counter"], b[5]["counter"] + np.asarray(rows, np.uint64))


def test_verification_non_finite_and_foreign_tokens(gpu):
    """A +inf logit is the whole distribution, -inf ones have no mass, a draft outside the vocabulary or outside the
    drafter's candidates is judged by P alone."""
    case("verify non-finite")
    rng = np.random.default_rng(7)
    for drafter in (True, False):
        b = batch(rng, 1200, [4, 4, 4, 4], [(0.8, 40, 0.95), (1.0, 1024, 1.0)], drafter)
        logits, dl, toks = b[0], b[1], b[2]
        logits[0, 700] = np.inf
        logits[1, 30:] = -np.inf
        logits[4, :] = -np.inf
        logits[5, ::2] = -np.inf
        toks[9], toks[10], toks[13] = -1, 1200, int(np.argmin(logits[12]))
        if drafter:
            dl[2, 11] = np.inf
            dl[6, :] = -np.inf
        out, n, _, _ = run(gpu, *b)
        eo, en = verify(*b)
        assert np.array_equal(n, en) and np.array_equal(out, eo)


def test_verification_draws_the_targets_distribution(gpu):
    """One draft of a drafter that is far off, many times: the first token's frequencies are the target's P.  With N
    draws each frequency is within 5 sqrt(p (1 - p) / N) of p but for odds of 1e-6 a token."""
    case("verify frequencies")
    rng = np.random.default_rng(8)
    V, N = 12, 20000
    l = (rng.standard_normal(V) * 1.2).astype(np.float32)
    d = (rng.standard_normal(V) * 1.2).astype(np.float32)
    ids, p = ranked(l, 1.0, 9, 1.0)
    qi, q = ranked(d, 1.0, 9, 1.0)
    B = 10000
    cnt = np.zeros(V)
    for _ in range(N // B):
        logits, dl = np.tile(l, (2 * B, 1)), np.tile(d, (2 * B, 1))
        toks = np.zeros(2 * B, np.int32)
        toks[1::2] = rng.choice(qi, B, p=q)
        params = np.zeros(B, PARAM_DT)
        params["temperature"], params["top_k"], params["top_p"] = 1.0, 9, 1.0
        out, n, _, _ = run(gpu, logits, dl, toks, np.arange(0, 2 * B + 1, 2).astype(np.int32),
                           rng.random(2 * B).astype(np.float32), params)
        cnt += np.bincount(out[::2], minlength=V)
    full = np.zeros(V)
    full[ids] = p
    assert np.all(np.abs(cnt / N - full) <= 5 * np.sqrt(full * (1 - full) / N))


def test_verification_replayed(gpu):
    """Captured once, replayed with other inputs and eager calls between."""
    case("verify graph")
    rng = np.random.default_rng(9)
    V, rows = 9000, [3, 1, 4]
    first = batch(rng, V, rows, SETTINGS, True)
    D = dr.DevTensor.from_host
    l, d, t, s, u, p = (D(x, gpu) for x in first[:5] + (first[5].view(np.uint8),))
    o, n = dr.DevTensor.empty((8,), np.int32, gpu), dr.DevTensor.empty((3,), np.int32, gpu)
    ws = dr.DevTensor.empty((dr.verify_drafts_workspace_size(8, V, True),), np.uint8, gpu)
    gpu.sync()
    call("lt_graph_begin", gpu.handle)
    dr.verify_drafts_into(l, t, s, u, p, o, n, ws, draft_logits=d)
    g = ctypes.c_void_p()
    call("lt_graph_end", gpu.handle, ctypes.byref(g))
    for _ in range(4):
        b = batch(rng, V, rows, SETTINGS, True)
        for dst, src in zip((l, d, t, u), (b[0], b[1], b[2], b[4])):
            dst.upload(src)
        call("lt_graph_launch", gpu.handle, g)
        out, cnt = o.to_host(), n.to_host()
        eo, en = verify(*b)
        assert np.array_equal(cnt, en) and np.array_equal(out, eo)
        dr.verify_drafts_into(l, t, s, u, p, o, n, ws, draft_logits=None)
        assert np.array_equal(o.to_host(), verify(b[0], None, *b[2:])[0])
    call("lt_graph_free", g)
    for x in (l, d, t, s, u, p, o, n, ws):
        x.free()


def test_verification_rows_behind_the_last_sequence(gpu):
    case("verify rows behind")
    rng = np.random.default_rng(10)
    logits, dl, toks, start, u, params = batch(rng, 700, [3, 2, 4], SETTINGS, True)
    start = start[:3]                                   # the last sequence's rows belong to nobody
    out, n, _, _ = run(gpu, logits, dl, toks, start, u, params[:2])
    eo, en = verify(logits[:5], dl[:5], toks[:5], start, u[:5], params[:2])
    assert np.array_equal(n, en) and np.array_equal(out[:5], eo) and np.all(out[5:] == -9)


def test_verification_no_rows(gpu):
    case("verify no rows")
    n = dr.DevTensor.from_host(np.full(2, -9, np.int32), gpu)
    s = dr.DevTensor.zeros((3,), np.int32, gpu)
    z = dr.DevTensor.zeros((64,), np.uint8, gpu)
    call("lt_verify_drafts", gpu.handle, z.vp, None, z.vp, s.vp, z.vp, z.vp, 2, 0, 100, z.vp, n.vp, None, z.vp, 0)
    assert np.array_equal(n.to_host(), [0, 0])
    for t in (n, s, z):
        t.free()
