"""The paged cache's kernels (lt_paged.hip) against plain float64: the append's rows bit for bit against the contiguous
append, attention over head layouts, page sizes, chunk lengths from none to long, windows, splits, poisoned masked
places, bad pages, pools past 4 GiB, captured graphs, and a run of append, attention and length update as they are used."""
import ctypes

import numpy as np
import pytest

from llamatov_amd import engine as dr
from llamatov_amd._lib import LT_KV_F16, LT_KV_F32, call

pytestmark = pytest.mark.gpu


def case(msg):
    print(f"[gpu-case] {msg}", flush=True)


class Batch:
    """A packed batch over a paged cache whose pools hold `fill` wherever no sequence's position lies."""

    def __init__(self, gpu, news, pasts, nh, nkv, hd, page, kv, seed=0, fill=None, extra=0, spread=1.0, T=None,
                 vals=None):
        self.gpu, self.news, self.pasts, self.nh, self.nkv, self.hd, self.page = gpu, news, pasts, nh, nkv, hd, page
        self.kv_dtype = LT_KV_F16 if kv == "f16" else LT_KV_F32
        self.np_dt = np.float16 if kv == "f16" else np.float32
        rng = np.random.default_rng(seed)
        self.rng = rng
        need = [-(-(p + n) // page) for p, n in zip(pasts, news)]
        n_pages = sum(need) + 2
        self.K = [(rng.standard_normal((p + n, nkv, hd)) * spread).astype(self.np_dt) for p, n in zip(pasts, news)]
        self.V = [rng.standard_normal((p + n, nkv, hd)).astype(self.np_dt) for p, n in zip(pasts, news)]
        if vals is not None:
            vals(self)
        fill = np.nan if fill is None else fill
        kp = np.full((n_pages, nkv, page, hd), fill, self.np_dt)
        vp = np.full((n_pages, nkv, page, hd), fill, self.np_dt)
        order = rng.permutation(n_pages)
        self.table = np.full((len(news), max(need + [1]) + 1), -1, np.int32)
        at = 0
        for b, (p, n) in enumerate(zip(pasts, news)):
            self.table[b, :need[b]] = order[at:at + need[b]]
            at += need[b]
            for t in range(p + n):
                pg = self.table[b, t // page]
                kp[pg, :, t % page] = self.K[b][t]
                vp[pg, :, t % page] = self.V[b][t]
        self.T = sum(news)
        self.rows = self.T if T is None else T
        self.q_stride = nh * hd + extra
        self.q = (rng.standard_normal((self.rows, self.q_stride)) * spread).astype(np.float32)
        self.start = np.cumsum([0] + list(news)).astype(np.int32)
        raw = np.uint16 if kv == "f16" else np.float32
        D = dr.DevTensor.from_host
        self.dk, self.dv, self.dt = D(kp.view(raw), gpu), D(vp.view(raw), gpu), D(self.table, gpu)
        self.kv = dr.PagedKV(self.dk, self.dv, self.dt, self.kv_dtype)
        self.dq, self.ds, self.dl = D(self.q, gpu), D(self.start, gpu), D(np.asarray(pasts, np.int32), gpu)
        self.out = D(np.full((self.rows, nh * hd), -7.0, np.float32), gpu)
        self.err = dr.DevTensor.zeros((1,), np.int32, gpu)
        self.scale = hd ** -0.5

    def attend(self, window=0, max_q=None, max_len=None):
        max_q = max(self.news) if max_q is None else max_q
        max_len = max(p + n for p, n in zip(self.pasts, self.news)) if max_len is None else max_len
        n = dr.attn_paged_workspace_size(self.rows, len(self.news), self.nh, self.kv, max_q, max_len)
        ws = dr.DevTensor.from_host(np.full(max(n, 16), 0xFF, np.uint8), self.gpu)   # NaN wherever nothing is written
        dr.attn_paged_into(self.dq, self.ds, self.dl, self.kv, self.nh, self.scale, self.out, max_q=max_q,
                           max_len=max_len, window=window, ws=ws, err=self.err)
        got = self.out.to_host()
        ws.free()
        return got

    def expect(self, window=0):
        """(the formula in float64, the bound of each row's error).

        Scores: hd products and sums in binary32, q taken in two binary16 terms (2^-22), the product with scale and the
        exponential's argument rounded: |ds| <= ((hd + 8) 2^-24 + 2^-21) scale sum |q||k| + 2^-22 |s|.  A weight is then
        off by |ds| + 2^-22 (the exponential, its two terms) of itself, the two sums of L terms by (L + 16) 2^-24."""
        out = np.zeros((self.rows, self.nh, self.hd))
        tol = np.zeros((self.rows, self.nh, 1))
        rep = self.nh // self.nkv
        for b, (p, n) in enumerate(zip(self.pasts, self.news)):
            K, V = self.K[b].astype(np.float64), self.V[b].astype(np.float64)
            for i in range(n):
                r = self.start[b] + i
                lo = max(0, p + i + 1 - window) if window else 0
                q = self.q[r, :self.nh * self.hd].astype(np.float64).reshape(self.nkv, rep, self.hd)
                k, v = K[lo:p + i + 1].transpose(1, 2, 0), V[lo:p + i + 1].transpose(1, 0, 2)
                s = q @ k * self.scale
                w = np.exp(s - s.max(-1, keepdims=True))
                z = w.sum(-1, keepdims=True)
                out[r] = (w @ v / z).reshape(self.nh, self.hd)
                sa = (np.abs(q) @ np.abs(k)).max(-1, keepdims=True) * self.scale
                ds = ((self.hd + 8) * 2.0 ** -24 + 2.0 ** -21) * sa + 2.0 ** -22 * np.abs(s).max(-1, keepdims=True)
                va = (w @ np.abs(v) / z).max(-1, keepdims=True)
                rel = 2 * (np.expm1(ds) + 2.0 ** -22) + 2 * (p + i + 17) * 2.0 ** -24
                tol[r] = (rel * va).reshape(self.nh, 1)
        return out.reshape(self.rows, -1), np.broadcast_to(tol, (self.rows, self.nh, self.hd)).reshape(self.rows, -1)

    def check(self, window=0, **kw):
        got = self.attend(window, **kw)
        exp, tol = self.expect(window)
        assert np.all(got[self.T:] == -7.0), "rows behind the last sequence were written"
        bad = ~(np.abs(got[:self.T] - exp[:self.T]) <= tol[:self.T])
        if bad.any():
            r, c = np.argwhere(bad)[0]
            raise AssertionError(f"{bad.sum()} of {bad.size} off, first row {r} head {c // self.hd} dim {c % self.hd}: "
                                 f"{got[r, c]} for {exp[r, c]} (+-{tol[r, c]})")
        assert int(self.err.to_host()[0]) == 0
        return got

    def free(self):
        for t in (self.dk, self.dv, self.dt, self.dq, self.ds, self.dl, self.out, self.err):
            t.free()


GEOMETRIES = [(14, 2, 64), (8, 2, 128), (4, 4, 40), (6, 1, 96), (4, 2, 256), (4, 1, 8), (2, 1, 136), (32, 1, 64)]


@pytest.mark.parametrize("kv", ["f16", "f32"])
@pytest.mark.parametrize("nh,nkv,hd", GEOMETRIES)
def test_attention_geometries(gpu, nh, nkv, hd, kv):
    for page, news, pasts in ((16, [1], [0]), (16, [1, 0, 5, 1], [61, 9, 0, 200]), (8, [3, 70], [130, 33])):
        case(f"attention {nh}/{nkv}/{hd} {kv} page {page} news {news} pasts {pasts}")
        b = Batch(gpu, news, pasts, nh, nkv, hd, page, kv, seed=hd + page)
        b.check()
        b.free()


@pytest.mark.parametrize("kv", ["f16", "f32"])
@pytest.mark.parametrize("page", [1, 2, 16, 64, 512])
def test_attention_page_sizes(gpu, page, kv):
    case(f"attention page {page} {kv}")
    b = Batch(gpu, [4, 33, 1], [67, 0, 129], 8, 2, 64, page, kv, seed=page)
    b.check()
    b.free()


@pytest.mark.parametrize("kv", ["f16", "f32"])
@pytest.mark.parametrize("n", [1, 2, 4, 5, 9, 16, 17, 31, 64, 65, 129])
def test_attention_chunk_lengths(gpu, n, kv):
    for past in (0, 1, 63, 300):
        case(f"attention chunk {n} over {past} {kv}")
        b = Batch(gpu, [n], [past], 8, 2, 128, 16, kv, seed=n * 7 + past)
        b.check()
        b.free()


@pytest.mark.parametrize("kv", ["f16", "f32"])
@pytest.mark.parametrize("window", [1, 2, 15, 64, 100])
def test_attention_windows(gpu, window, kv):
    """A window that ends inside tiles and pages; what lies before it is poison, and its pages are given back."""
    for news, pasts in (([1, 3, 1], [0, 250, 40]), ([80, 7], [190, 0])):
        case(f"attention window {window} {kv} {news}")

        def poison(b):
            for i, p in enumerate(b.pasts):
                b.K[i][:max(0, p + 1 - window)] = np.nan
                b.V[i][:max(0, p + 1 - window)] = np.inf
        b = Batch(gpu, news, pasts, 8, 2, 64, 16, kv, seed=window, vals=poison)
        for i, p in enumerate(pasts):
            b.table[i, :max(0, p + 1 - window) // 16] = -1
        b.dt.upload(b.table)
        exp, tol = b.expect(window)
        got = b.attend(window)
        assert np.all(np.abs(got - exp) <= tol) and int(b.err.to_host()[0]) == 0
        b.free()


def test_attention_split_windows(gpu):
    """Windows over long contexts: the workspace of the whole context serves every window."""
    for news, pasts in (([5, 1], [3000, 2600]), ([40, 17], [4500, 2600])):
        b = Batch(gpu, news, pasts, 8, 2, 64, 32, "f16", seed=21)
        for window in (300, 700, 1000, 2047, 2999, 5000):
            case(f"attention split window {window} {news}")
            b.check(window=window)
        b.free()


@pytest.mark.parametrize("kv", ["f16", "f32"])
@pytest.mark.parametrize("news,pasts,max_len", [([1], [5000], None), ([5, 1, 2], [3000, 1, 900], None),
                                                ([70], [2500], None), ([1, 1], [4097, 130], 1), ([40], [2000], 0),
                                                ([90, 3], [3900, 100], None)])
def test_attention_splits(gpu, news, pasts, max_len, kv):
    """Long contexts of few rows, and host bounds that are wrong or not known."""
    case(f"attention long {news} {pasts} {max_len} {kv}")
    b = Batch(gpu, news, pasts, 8, 2, 128, 32, kv, seed=9)
    first = b.check(max_len=max_len, max_q=0 if max_len == 0 else None)
    again = b.check(max_len=max_len, max_q=0 if max_len == 0 else None)
    assert np.array_equal(first, again)      # no order of arrival in the result
    if max_len is None:
        b.check(max_q=1, max_len=100000)
    b.free()


@pytest.mark.parametrize("kv", ["f16", "f32"])
@pytest.mark.parametrize("nh,nkv,hd", [(14, 2, 64), (8, 2, 128), (6, 1, 96), (4, 1, 40), (4, 2, 256)])
def test_attention_long_chunks(gpu, nh, nkv, hd, kv):
    """Many rows over contexts long enough for the widest tiles, with and without a window."""
    b = Batch(gpu, [75, 1, 40], [3650, 17, 2000], nh, nkv, hd, 32, kv, seed=hd)
    for window in (0, 3600, 700):
        case(f"attention long chunks {nh}/{nkv}/{hd} {kv} window {window}")
        b.check(window=window)
    b.free()


def test_attention_large_batch(gpu):
    case("attention 150 sequences of unequal lengths")
    rng = np.random.default_rng(3)
    news = [int(v) for v in rng.integers(0, 4, 150)]
    pasts = [int(v) for v in rng.integers(0, 90, 150)]
    news[10], news[77] = 60, 45
    b = Batch(gpu, news, pasts, 4, 2, 64, 16, "f16", seed=4, T=sum(news) + 9, extra=12)
    b.check()
    b.free()


@pytest.mark.parametrize("kv", ["f16", "f32"])
def test_attention_many_drafts(gpu, kv):
    """More workgroups of up to 32 rows than CUs, with and without splits."""
    rng = np.random.default_rng(5)
    for B, ctx in ((70, 150), (35, 900)):
        case(f"attention {B} chunks of drafts over up to {ctx} {kv}")
        news = [int(v) for v in rng.integers(1, 9, B)]
        b = Batch(gpu, news, [int(v) for v in rng.integers(0, ctx, B)], 16, 4, 64, 16, kv, seed=B)
        b.check(max_q=8)
        b.free()


def test_attention_strides(gpu):
    """q rows that are not 16-byte aligned, and rows behind the last sequence."""
    for extra in (1, 3, 8, 130):
        case(f"attention q_stride + {extra}")
        b = Batch(gpu, [3, 2], [20, 50], 4, 2, 64, 16, "f16", seed=extra, extra=extra, T=9)
        b.check()
        b.free()


@pytest.mark.parametrize("kv", ["f16", "f32"])
def test_attention_peaked_and_flat(gpu, kv):
    """Scores over hundreds (one key takes all) and equal scores; queries of very different sizes."""
    case(f"attention peaked {kv}")
    b = Batch(gpu, [40, 2], [700, 90], 8, 2, 64, 16, kv, seed=2, spread=8.0)
    b.check()
    b.free()

    def zero(b):
        for k in b.K:
            k[:] = 0
    b = Batch(gpu, [40, 2], [700, 90], 8, 2, 64, 16, kv, seed=2, vals=zero)
    b.check()
    b.free()
    b = Batch(gpu, [6], [50], 8, 2, 64, 16, kv, seed=2)
    b.q *= np.array([1e-30, 1e-6, 1.0, 0.0, 30.0, 1e-42], np.float32)[:, None]
    b.dq.upload(b.q)
    b.check()
    b.free()


@pytest.mark.parametrize("kv", ["f16", "f32"])
@pytest.mark.parametrize("scale", [-0.2, 0.0, 3.0])
def test_attention_scales(gpu, scale, kv):
    """A negative scale turns the order of the keys round, zero makes every weight the same."""
    case(f"attention scale {scale} {kv}")
    b = Batch(gpu, [3, 40], [700, 20], 4, 2, 64, 16, kv, seed=6)
    b.scale = scale
    got = b.attend()
    k, b.scale = b.K, abs(scale)
    b.K = [x * np.sign(scale).astype(x.dtype) for x in b.K]
    exp, tol = b.expect()
    assert np.all(np.abs(got - exp) <= tol)
    b.free()


@pytest.mark.parametrize("n", [2, 40])
def test_attention_large_fp32_values(gpu, n):
    """Values near the largest binary32: the result is a mean of them, and no step of the way is larger."""
    case(f"attention large values, chunk of {n}")

    def large(b):
        b.V[0] *= np.float32(2.0 ** 115)              # to 2^117, 400 of them, and a weight of 2^-8 at most each step
    b = Batch(gpu, [n], [400], 4, 2, 64, 16, "f32", seed=7, vals=large)
    b.check()
    b.free()


@pytest.mark.parametrize("kv", ["f16", "f32"])
@pytest.mark.parametrize("n,past", [(4, 33), (20, 33), (90, 33), (90, 3800)])
def test_attention_masked_infinities(gpu, n, past, kv):
    """A later token's K and V of infinities and NaN do not reach the rows before it; the rows that attend it follow
    the formula."""
    case(f"attention masked infinities, chunk of {n} over {past}, {kv}")
    at = past + n - 2

    def spoil(b):
        b.V[0][at, 0, 3] = np.inf
        b.V[0][at, 1, 5] = np.nan
        b.V[0][at + 1, 0, 3] = -np.inf
        b.K[0][at + 1, 1] = np.nan
    b = Batch(gpu, [n], [past], 8, 2, 64, 16, kv, seed=n, vals=spoil)
    got = b.attend().reshape(n, 2, 4, 64)
    with np.errstate(all="ignore"):
        exp, tol = b.expect()
    exp, tol = exp.reshape(n, 2, 4, 64), tol.reshape(n, 2, 4, 64)
    assert np.all(np.abs(got - exp)[:n - 2] <= tol[:n - 2])
    row = got[n - 2]                                   # attends position `at`, not at + 1
    assert np.all(row[0, :, 3] == np.inf) and np.all(np.isnan(row[1, :, 5]))
    keep = np.ones((2, 64), bool)
    keep[0, 3] = keep[1, 5] = False
    for h in range(2):
        d = keep[h]
        assert np.all(np.isfinite(row[h][:, d]))
    last = got[n - 1]
    assert np.all(np.isnan(last[0, :, 3])) and np.all(np.isnan(last[1]))
    d = keep[0]
    assert np.all(np.isfinite(last[0][:, d]))
    b.free()


@pytest.mark.parametrize("kv", ["f16", "f32"])
@pytest.mark.parametrize("n,past", [(1, 300), (6, 300), (40, 300), (90, 300), (90, 3700)])
def test_attention_attended_infinities(gpu, n, past, kv):
    """Infinities among the values and keys that every row attends, deep inside the context: the formula's infinity, NaN
    where two of them cancel, nothing else touched; a key of -inf for positive queries has no weight."""
    case(f"attention attended infinities, chunk of {n} over {past}, {kv}")

    def spoil(b):
        b.V[0][100, 0, 3] = np.inf
        b.V[0][101, 0, 4] = -np.inf
        b.V[0][102, 0, 5], b.V[0][103, 0, 5] = np.inf, -np.inf
        b.V[0][104, 1, 6] = np.nan
        b.K[0][200] = -np.inf
        b.V[0][200] = 1000.0
    b = Batch(gpu, [n], [past], 8, 2, 64, 16, kv, seed=n, vals=spoil)
    b.q[:] = np.abs(b.q) + 0.25
    b.q[:, 1] = 0.5                                    # exact in few bits: the second term has nothing left
    b.dq.upload(b.q)
    got = b.attend().reshape(n, 2, 4, 64)
    assert np.all(got[:, 0, :, 3] == np.inf) and np.all(got[:, 0, :, 4] == -np.inf)
    assert np.all(np.isnan(got[:, 0, :, 5])) and np.all(np.isnan(got[:, 1, :, 6]))
    for i, d in ((100, 3), (101, 4), (102, 5), (103, 5)):
        b.V[0][i, 0, d] = 0
    b.V[0][104, 1, 6] = 0
    with np.errstate(all="ignore"):
        b.K[0][200] = -60000.0                         # no weight either
        exp, _ = b.expect()
        b.K[0][200] = 0
        _, tol = b.expect()
    exp, tol = exp.reshape(n, 2, 4, 64), tol.reshape(n, 2, 4, 64)
    keep = np.ones((2, 64), bool)
    keep[0, 3:6] = keep[1, 6] = False
    for h in range(2):
        d = keep[h]
        assert np.all(np.abs(got - exp)[:, h][..., d] <= tol[:, h][..., d])
    b.free()


@pytest.mark.parametrize("kv", ["f16", "f32"])
def test_attention_all_scores_minus_infinity(gpu, kv):
    """Keys of -inf for a positive query: exp(-inf - -inf) is NaN, as the formula has it; one finite key wins alone."""
    case(f"attention keys of -inf {kv}")

    def spoil(b):
        b.K[0][:] = -np.inf
        b.K[1][:] = -np.inf
        b.K[1][3] = 0.0
    b = Batch(gpu, [1, 1], [20, 20], 2, 1, 64, 16, kv, seed=1, vals=spoil)
    b.q[:] = np.abs(b.q) + 0.5
    b.dq.upload(b.q)
    got = b.attend()
    assert np.all(np.isnan(got[0]))
    assert np.array_equal(got[1], np.tile(b.V[1][3].astype(np.float32).reshape(-1), 2))
    b.free()


@pytest.mark.parametrize("kv", ["f16", "f32"])
def test_attention_bad_pages(gpu, kv):
    """Page ids outside the pool read as zero rows and set the flag; a length past the table's row is cut there."""
    for news, pasts in (([1, 2], [40, 40]), ([70, 2], [40, 40])):
        case(f"attention bad pages {kv} {news}")
        b = Batch(gpu, news, pasts, 4, 2, 64, 16, kv, seed=5)
        n_pages = b.dk.shape[0]
        t = b.table.copy()
        t[0, 1] = n_pages
        t[1, 0] = -3
        b.dt.upload(t)
        got = b.attend()
        assert int(b.err.to_host()[0]) == 1
        b.K[0][16:32] = 0
        b.V[0][16:32] = 0
        b.K[1][:16] = 0
        b.V[1][:16] = 0
        exp, tol = b.expect()
        assert np.all(np.abs(got - exp) <= tol)
        b.free()


@pytest.mark.parametrize("kv", ["f16", "f32"])
def test_attention_length_past_the_table(gpu, kv):
    """Rows past the table's row attend what it holds, and set the flag."""
    for n in (1, 30):
        case(f"attention past the table {kv} chunk {n}")
        b = Batch(gpu, [n, 2], [40, 40], 4, 2, 64, 16, kv, seed=5, fill=0.5)
        b.table[0][b.table[0] < 0] = 0
        b.dt.upload(b.table)
        for length in (b.table.shape[1] * 16, 2 ** 31 - 1):
            b.dl.upload(np.asarray([length, 40], np.int32))
            b.gpu.fill(b.err.ptr, 0, 4)
            got = b.attend()
            assert int(b.err.to_host()[0]) == 1
            rows = []
            for pool in (b.dk, b.dv):
                v = pool.to_host().view(b.np_dt)[b.table[0]]             # [pages][nkv][page][hd]
                rows.append(v.transpose(0, 2, 1, 3).reshape(-1, 2, 64).astype(np.float64))
            s = np.einsum("rghd,tgd->rght", b.q[:n].astype(np.float64).reshape(n, 2, 2, 64), rows[0]) / 8
            w = np.exp(s - s.max(-1, keepdims=True))
            exp = np.einsum("rght,tgd->rghd", w / w.sum(-1, keepdims=True), rows[1]).reshape(n, -1)
            exp2, tol = b.expect()                                        # sequence 1's rows, and the bound
            assert np.all(np.abs(got[n:] - exp2[n:]) <= tol[n:])
            # the bound of expect() grows with the positions, of which there are at most twice as many here
            assert np.all(np.abs(got[:n] - exp) <= 4 * tol[:n].max())
        b.free()


def test_attention_pool_past_4gib(gpu):
    """Offsets in the pools past 2^32 bytes and 2^31 elements."""
    nkv, page, hd = 8, 64, 128
    n_pages = (5 << 30) // (nkv * page * hd * 2)
    case(f"attention over pools of {n_pages} pages")
    k = dr.DevTensor.empty((n_pages, nkv, page, hd), np.uint16, gpu)
    v = dr.DevTensor.empty((n_pages, nkv, page, hd), np.uint16, gpu)
    table = np.array([[n_pages - 1, 0, n_pages - 7, n_pages // 2 + 1]], np.int32)
    dt = dr.DevTensor.from_host(table, gpu)
    kv = dr.PagedKV(k, v, dt, LT_KV_F16)
    small = Batch(gpu, [5], [190], 8, nkv, hd, page, "f16", seed=11)
    full = (small.pasts[0] + small.news[0] + page - 1) // page
    pk = small.dk.to_host()
    pv = small.dv.to_host()
    for j in range(full):
        off = int(table[0, j]) * nkv * page * hd * 2
        gpu.h2d(k.ptr + off, pk[small.table[0, j]])
        gpu.h2d(v.ptr + off, pv[small.table[0, j]])
    exp = small.check()
    small.kv = kv
    assert np.array_equal(small.attend(), exp)
    # the append writes there too
    nq = (8 + 2 * nkv) * hd
    qkv = small.rng.standard_normal((5, nq)).astype(np.float32)
    dqkv, qo = dr.DevTensor.from_host(qkv, gpu), dr.DevTensor.empty((5, 8 * hd), np.float32, gpu)
    fr = dr.DevTensor.from_host(dr.rope_freqs(hd, 5e5), gpu)
    dr.rope_append_paged_into(dqkv, qo, small.ds, small.dl, 8, fr, kv)
    gpu.sync()
    row = np.empty(hd, np.float16)
    gpu.d2h(row, v.ptr + ((int(table[0, 191 // page]) * nkv + 7) * page + 191 % page) * hd * 2)
    assert np.array_equal(row, qkv[1, -hd:].astype(np.float16))
    for t in (k, v, dt, dqkv, qo, fr):
        t.free()
    small.free()


# ---- RoPE and append ---------------------------------------------------------------------------
def contiguous_append(gpu, qkv, past, nh, nkv, hd, freqs, kv_dtype, maxt):
    """lt_rope_append_batch of one sequence: q rows and cache rows."""
    n = len(qkv)
    raw = np.uint16 if kv_dtype == LT_KV_F16 else np.float32
    x = dr.DevTensor.from_host(qkv, gpu)
    k, v = dr.DevTensor.zeros((maxt, nkv, hd), raw, gpu), dr.DevTensor.zeros((maxt, nkv, hd), raw, gpu)
    ln = dr.DevTensor.from_host(np.array([past], np.int32), gpu)
    call("lt_rope_append_batch", gpu.handle, x.vp, n, qkv.shape[1], ln.vp, nh, nkv, hd, freqs.vp, k.vp, v.vp, maxt,
         kv_dtype)
    got = x.to_host()[:, :nh * hd], k.to_host()[past:past + n], v.to_host()[past:past + n]
    for t in (x, k, v, ln):
        t.free()
    return got


@pytest.mark.parametrize("kv", ["f16", "f32"])
@pytest.mark.parametrize("nh,nkv,hd", [(14, 2, 64), (8, 2, 128), (4, 4, 40), (2, 1, 256), (4, 1, 8)])
@pytest.mark.parametrize("page,news,pasts", [(16, [1], [0]), (16, [1, 0, 70, 3], [130, 7, 0, 15]), (1, [5, 2], [0, 9]),
                                             (64, [129, 1], [63, 4000])])
def test_append_matches_the_contiguous_append(gpu, page, news, pasts, nh, nkv, hd, kv):
    case(f"append {nh}/{nkv}/{hd} {kv} page {page} news {news} pasts {pasts}")
    b = Batch(gpu, news, pasts, nh, nkv, hd, page, kv, seed=1, fill=3.0, T=sum(news) + 2)
    width = (nh + 2 * nkv) * hd
    qkv = b.rng.standard_normal((b.rows, width + 5)).astype(np.float32) * 3
    freqs = dr.DevTensor.from_host(dr.rope_freqs(hd, 1e4), gpu)
    pk, pv = b.dk.to_host(), b.dv.to_host()
    for in_place in (False, True):
        x = dr.DevTensor.from_host(qkv, gpu)
        qo = x if in_place else dr.DevTensor.from_host(np.full((b.rows, nh * hd + 3), -7.0, np.float32), gpu)
        dr.rope_append_paged_into(x, qo, b.ds, b.dl, nh, freqs, b.kv, b.err)
        gk, gv, gq, gx = b.dk.to_host(), b.dv.to_host(), qo.to_host(), x.to_host()
        ek, ev = pk.copy(), pv.copy()
        for s, (n, p) in enumerate(zip(news, pasts)):
            if not n:
                continue
            eq, rk, rv = contiguous_append(gpu, qkv[b.start[s]:b.start[s + 1]], p, nh, nkv, hd, freqs, b.kv_dtype,
                                           p + n)
            assert np.array_equal(gq[b.start[s]:b.start[s + 1], :nh * hd].view(np.uint32), eq.view(np.uint32))
            for t in range(n):
                pg, sl = b.table[s, (p + t) // page], (p + t) % page
                ek[pg, :, sl], ev[pg, :, sl] = rk[t], rv[t]
        assert np.array_equal(gk, ek) and np.array_equal(gv, ev)      # and nothing else in the pools changed
        assert np.array_equal(gx[:, nh * hd:], qkv[:, nh * hd:])      # q|k|v's own k and v are left
        assert np.array_equal(gx[b.T:], qkv[b.T:])
        if not in_place:
            assert np.all(gq[b.T:] == -7.0) and np.all(gq[:, nh * hd:] == -7.0) and np.array_equal(gx, qkv)
            qo.free()
        x.free()
    assert int(b.err.to_host()[0]) == 0
    freqs.free()
    b.free()


def test_append_bad_pages(gpu):
    """Positions without a page are not stored and set the flag; the others are."""
    case("append bad pages")
    b = Batch(gpu, [20, 2], [10, 5], 4, 2, 64, 16, "f32", seed=1, fill=3.0)
    t = b.table.copy()
    t[0, 1] = b.dk.shape[0] + 5
    b.dt.upload(t)
    qkv = b.rng.standard_normal((22, 8 * 64)).astype(np.float32)
    x, qo = dr.DevTensor.from_host(qkv, gpu), dr.DevTensor.empty((22, 4 * 64), np.float32, gpu)
    freqs = dr.DevTensor.from_host(dr.rope_freqs(64, 1e4), gpu)
    pv = b.dv.to_host()
    dr.rope_append_paged_into(x, qo, b.ds, b.dl, 4, freqs, b.kv, b.err)
    gv = b.dv.to_host()
    assert int(b.err.to_host()[0]) == 1
    ev = pv.copy()
    for r in range(6):
        ev[t[0, 0], :, 10 + r] = qkv[r, 6 * 64:].reshape(2, 64)
    for r in range(2):
        ev[t[1, 0], :, 5 + r] = qkv[20 + r, 6 * 64:].reshape(2, 64)
    assert np.array_equal(gv, ev)
    b.gpu.fill(b.err.ptr, 0, 4)
    b.dl.upload(np.array([b.table.shape[1] * 16 - 1, 2 ** 31 - 5], np.int32))   # past the table's row
    b.dt.upload(np.full_like(b.table, -1))
    dr.rope_append_paged_into(x, qo, b.ds, b.dl, 4, freqs, b.kv, b.err)
    assert int(b.err.to_host()[0]) == 1 and np.array_equal(b.dv.to_host(), gv)
    for v in (x, qo, freqs):
        v.free()
    b.free()


# ---- together, captured, replayed --------------------------------------------------------------
@pytest.mark.parametrize("kv", ["f16", "f32"])
def test_append_attend_advance_replayed(gpu, kv):
    """Append, attention and the length update of a batch captured once and replayed over growing contexts, with eager
    work between the replays, against the formula each time."""
    nh, nkv, hd, page = 8, 2, 64, 16
    case(f"append + attention graph {kv}")
    cache = dr.PagedKVCache(1, 40, page, nkv, hd, max_seqs=3, max_pages=16,
                            kv_dtype=LT_KV_F16 if kv == "f16" else LT_KV_F32, dev=gpu)
    news = [2, 0, 5]
    T, L = 7, cache.layers[0]
    start = dr.DevTensor.from_host(np.cumsum([0] + news).astype(np.int32), gpu)
    x = dr.DevTensor.empty((T, (nh + 2 * nkv) * hd), np.float32, gpu)
    q, out = dr.DevTensor.empty((T, nh * hd), np.float32, gpu), dr.DevTensor.empty((T, nh * hd), np.float32, gpu)
    freqs_h = dr.rope_freqs(hd, 1e4)
    freqs = dr.DevTensor.from_host(freqs_h, gpu)
    n = dr.attn_paged_workspace_size(T, 3, nh, L, 5, 256)
    ws, err = dr.DevTensor.empty((max(n, 16),), np.uint8, gpu), dr.DevTensor.zeros((1,), np.int32, gpu)
    for b in range(3):
        cache.reserve(b, 6 * max(news[b], 1))
    cache.set_lengths([0, 0, 0])
    gpu.sync()
    call("lt_graph_begin", gpu.handle)
    dr.rope_append_paged_into(x, q, start, cache.lens, nh, freqs, L, err)
    dr.attn_paged_into(q, start, cache.lens, L, nh, hd ** -0.5, out, max_q=5, max_len=256, ws=ws, err=err)
    call("lt_len_add_rows", gpu.handle, cache.lens.vp, start.vp, 3, 16 * page)
    g = ctypes.c_void_p()
    call("lt_graph_end", gpu.handle, ctypes.byref(g))
    rng = np.random.default_rng(8)
    K, V = [[] for _ in news], [[] for _ in news]
    dt = np.float16 if kv == "f16" else np.float32
    scratch = dr.DevTensor.empty((T, nh * hd), np.float32, gpu)
    for step in range(5):
        rows = rng.standard_normal((T, (nh + 2 * nkv) * hd)).astype(np.float32)
        x.upload(rows)
        before = cache.lengths()
        call("lt_graph_launch", gpu.handle, g)
        got = out.to_host()
        assert cache.lengths() == [a + b for a, b in zip(before, news)]
        assert int(err.to_host()[0]) == 0
        qh = q.to_host().reshape(T, nkv, nh // nkv, hd).astype(np.float64)
        r = 0
        for b, m in enumerate(news):
            for i in range(m):
                # the cached row as binary32 rope gives it, in the cache's type
                a = (np.float32(before[b] + i) * freqs_h).astype(np.float64)
                kk = rows[r, nh * hd:(nh + nkv) * hd].reshape(nkv, 2, hd // 2).astype(np.float64)
                kr = np.concatenate([kk[:, 0] * np.cos(a) - kk[:, 1] * np.sin(a),
                                     kk[:, 0] * np.sin(a) + kk[:, 1] * np.cos(a)], -1)
                K[b].append(kr.astype(np.float32).astype(dt).astype(np.float64))
                V[b].append(rows[r, (nh + nkv) * hd:].reshape(nkv, hd).astype(dt).astype(np.float64))
                s = qh[r] @ np.stack(K[b], -1).reshape(nkv, hd, -1) * hd ** -0.5
                w = np.exp(s - s.max(-1, keepdims=True))
                e = (w @ np.stack(V[b], 1) / w.sum(-1, keepdims=True)).reshape(-1)
                # a key rounded the other way moves a score by half a step of its type; the weights by that and no more
                step_k = (2.0 ** -11 if kv == "f16" else 2.0 ** -23) * np.abs(kr).max()
                ds = hd ** -0.5 * np.abs(qh[r]).sum(-1).max() * step_k + 1e-5
                assert np.abs(got[r] - e).max() <= 2 * np.expm1(ds) * np.abs(np.stack(V[b])).max()
                r += 1
        # eager work between the replays, over the same workspace
        dr.attn_paged_into(q, start, dr.DevTensor(cache.lens.ptr, (3,), np.int32, False, gpu), L, nh, 0.5, scratch,
                           max_q=5, max_len=256, ws=ws)
        gpu.sync()
    call("lt_graph_free", g)
    for t in (start, x, q, out, freqs, ws, err, scratch):
        t.free()
    cache.free()


def test_empty_calls(gpu):
    case("no rows")
    b = Batch(gpu, [0, 0], [5, 0], 4, 2, 64, 16, "f16")
    z = dr.DevTensor.empty((1, 4 * 64), np.float32, gpu)
    call("lt_attn_paged", gpu.handle, z.ptr, 256, 0, b.ds.ptr, b.dl.ptr, 2, 4, b.kv.desc, z.ptr, 0.1, 0, 0, 0, None, 0,
         None)
    b.free()
    b = Batch(gpu, [0, 0], [5, 0], 4, 2, 64, 16, "f16", T=3)
    b.check()
    b.free()
    z.free()


def test_len_add_rows(gpu):
    case("lt_len_add_rows")
    n = 300
    rng = np.random.default_rng(0)
    ln, add = rng.integers(0, 50, n).astype(np.int32), rng.integers(0, 9, n)
    start = np.cumsum([0] + list(add)).astype(np.int32)
    d, s = dr.DevTensor.from_host(ln, gpu), dr.DevTensor.from_host(start, gpu)
    call("lt_len_add_rows", gpu.handle, d.vp, s.vp, n, 52)
    assert np.array_equal(d.to_host(), np.minimum(ln + add, 52))
    d.free()
    s.free()


def test_two_contexts_at_once(gpu):
    """Calls of two contexts in flight together, each with its own workspace, give what they give alone."""
    case("two contexts")
    other = dr.Device(0)
    batches = [Batch(d, [5, 1, 40], [1500, 3000, 90], 8, 2, 128, 16, kv, seed=s)
               for d, kv, s in ((gpu, "f16", 1), (other, "f32", 2))]
    alone = [b.attend() for b in batches]
    ws = []
    for b in batches:
        n = dr.attn_paged_workspace_size(b.rows, 3, b.nh, b.kv, 40, 3001)
        ws.append(dr.DevTensor.empty((max(n, 16),), np.uint8, b.gpu))
        b.out.upload(np.full((b.rows, b.nh * b.hd), -7.0, np.float32))
    for _ in range(20):
        for b, w in zip(batches, ws):
            dr.attn_paged_into(b.dq, b.ds, b.dl, b.kv, b.nh, b.scale, b.out, max_q=40, max_len=3001, ws=w)
    for b, a in zip(batches, alone):
        assert np.array_equal(b.out.to_host(), a)
    for b, w in zip(batches, ws):
        w.free()
        b.free()
    call("lt_free_ctx", other.handle)


def test_shared_prefix_pages(gpu):
    """Two sequences whose first pages are the same ones."""
    case("shared pages")
    b = Batch(gpu, [3, 3], [64, 64], 4, 2, 64, 16, "f16", seed=3)
    t = b.table.copy()
    t[1, :4] = t[0, :4]
    b.dt.upload(t)
    b.K[1][:64], b.V[1][:64] = b.K[0][:64], b.V[0][:64]
    b.check()
    b.free()
