"""The paged cache's host side without a GPU: the refusals of the three entry points (arguments are checked before the
context), workspace sizes, and the page account of engine.PagedKVCache over a device that only keeps host copies."""
import ctypes

import numpy as np
import pytest

from llamatov_amd import _lib
from llamatov_amd import engine as dr
from llamatov_amd._lib import LT_KV_F16, LT_KV_F32, PagedKvDesc

P = ctypes.c_void_p
GOOD = dict(kc=4096, vc=8192, table=4, table_stride=8, n_pages=16, page=16, nkv=2, hd=64, kv_dtype=LT_KV_F16)


def desc(**kw):
    return PagedKvDesc(*{**GOOD, **kw}.values())


BAD_CACHES = [(dict(kc=0), "null pool"), (dict(vc=0), "null pool"), (dict(table=0), "null pool"),
              (dict(kc=4104), "aligned"), (dict(table=6), "aligned"), (dict(page=0), "power of two"),
              (dict(page=24), "power of two"), (dict(page=-16), "power of two"), (dict(n_pages=0), "n_pages"),
              (dict(table_stride=0), "table_stride"), (dict(page=1 << 20, table_stride=1 << 11), "2^30"),
              (dict(hd=12), "multiple of 8"), (dict(hd=264), "at most 256"), (dict(nkv=0), "nkv"),
              (dict(nkv=3), "multiple of nkv"), (dict(kv_dtype=2), "kv_dtype")]


def attn(kv, **kw):
    a = dict(q=16, q_stride=256, T=4, q_start=4, len=4, B=1, nh=4, out=16, scale=0.1, window=0, max_q=0, max_len=0, ws=0,
             n=0)
    a.update(kw)
    return _lib.raw("lt_attn_paged")(None, a["q"], a["q_stride"], a["T"], a["q_start"], a["len"], a["B"], a["nh"], kv,
                                     a["out"], a["scale"], a["window"], a["max_q"], a["max_len"], a["ws"], a["n"], None)


def append(kv, **kw):
    a = dict(qkv=16, row_stride=512, q_out=64, q_stride=256, T=4, q_start=4, len=4, B=1, nh=4, freqs=4)
    a.update(kw)
    return _lib.raw("lt_rope_append_paged")(None, a["qkv"], a["row_stride"], a["q_out"], a["q_stride"], a["T"],
                                            a["q_start"], a["len"], a["B"], a["nh"], a["freqs"], kv, None)


def verify(**kw):
    a = dict(logits=16, dl=16, toks=4, q_start=4, u=4, params=8, B=1, T=4, V=100, out=4, n_out=4, len=0, ws=16, n=1 << 30)
    a.update(kw)
    return _lib.raw("lt_verify_drafts")(None, a["logits"], a["dl"], a["toks"], a["q_start"], a["u"], a["params"], a["B"],
                                        a["T"], a["V"], a["out"], a["n_out"], a["len"], a["ws"], a["n"])


def refused(rc, text):
    assert rc == -1 and text in _lib.last_error(), (rc, _lib.last_error())


@pytest.mark.parametrize("bad,text", BAD_CACHES)
def test_bad_caches_are_refused(bad, text):
    refused(attn(desc(**bad)), text)
    refused(append(desc(**bad)), text)


def test_attention_refusals():
    for name in ("q", "out", "q_start", "len"):
        refused(attn(desc(), **{name: 0}), "null")
    refused(attn(None), "null cache descriptor")
    refused(attn(desc(), q_stride=255), "q_stride")
    refused(attn(desc(), T=-1), "T=-1")
    refused(attn(desc(), B=0), "B=0")
    refused(attn(desc(), window=-1), "window=-1")
    refused(attn(desc(), max_q=-1), "max_q=-1")
    refused(attn(desc(), max_len=-1), "max_len=-1")
    refused(attn(desc()), "null ctx")      # every argument before it is in order
    n = dr._lib.raw("lt_attn_paged_workspace_size")(1, 1, 4, desc(page=64, table_stride=512), 1, 32768)
    if n:
        kv = desc(page=64, table_stride=512)
        assert attn(kv, T=1, max_q=1, max_len=32768, ws=16, n=n - 1) == -3
        refused(attn(kv, T=1, max_q=1, max_len=32768, ws=0, n=n), "null workspace")
        refused(attn(kv, T=1, max_q=1, max_len=32768, ws=8, n=n), "aligned")
        refused(attn(kv, T=1, max_q=1, max_len=32768, ws=16, n=n), "null ctx")


def test_append_refusals():
    for name in ("qkv", "q_out", "q_start", "len", "freqs"):
        refused(append(desc(), **{name: 0}), "null")
    refused(append(desc(), row_stride=511), "row_stride")
    refused(append(desc(), q_stride=255), "q_stride")
    refused(append(desc(), T=-1), "T=-1")
    refused(append(desc(), B=0), "B=0")
    refused(append(desc(), q_out=16), "in place")
    refused(append(desc(), q_out=16, q_stride=512), "null ctx")
    refused(append(desc()), "null ctx")


def test_verification_refusals():
    for name in ("logits", "toks", "q_start", "params", "out", "n_out", "ws"):
        refused(verify(**{name: 0}), "null")
    refused(verify(B=0), "B=0")
    refused(verify(T=-1), "T=-1")
    refused(verify(T=32768), "T=32768")
    refused(verify(V=0), "V=0")
    refused(verify(V=262145), "V=262145")
    refused(verify(params=4), "aligned")
    refused(verify(ws=4), "aligned")
    refused(verify(), "null ctx")
    refused(verify(dl=0, u=0), "null ctx")
    need = _lib.raw("lt_verify_drafts_workspace_size")(4, 100, 1)
    assert verify(n=need - 1) == -3
    refused(verify(T=0, ws=0, n=0), "null ctx")     # no rows need no workspace
    refused(verify(n=need), "null ctx")


def test_len_add_rows_refusals():
    f = _lib.raw("lt_len_add_rows")
    refused(f(None, 0, 4, 1, 8), "null")
    refused(f(None, 4, 4, 0, 8), "B=0")
    refused(f(None, 4, 4, 1, 0), "maxt=0")
    refused(f(None, 4, 4, 1, 8), "null ctx")


def test_workspace_sizes():
    v = _lib.raw("lt_verify_drafts_workspace_size")
    assert v(0, 100, 1) == 0 and v(4, 262145, 1) == 0 and v(-1, 100, 0) == 0
    assert v(4, 151936, 0) < v(4, 151936, 1) < v(320, 151936, 1)
    a = _lib.raw("lt_attn_paged_workspace_size")
    assert a(0, 1, 4, desc(), 0, 0) == 0
    assert a(1, 1, 4, desc(hd=12), 0, 0) == 0      # refused geometries have no size


def test_workspace_serves_every_window():
    """The size asked for without a window is enough with any (arithmetic of the launch plan)."""
    need = _lib.raw("lt_attn_paged_workspace_size")
    run = _lib.raw("lt_attn_paged")
    for page, stride in ((16, 300), (64, 512)):
        for f16 in (LT_KV_F16, LT_KV_F32):
            for nh, nkv, hd in ((8, 2, 64), (32, 8, 128), (4, 1, 256)):
                kv = PagedKvDesc(4096, 4096, 4, stride, 100, page, nkv, hd, f16)
                for T in (1, 4, 9, 30, 100, 700, 3000):
                    for L in (1, 300, 4000, 30000):
                        n = need(T, 2, nh, kv, T, L)
                        for window in (1, 100, 1000, 3499, 3600, 20000):
                            rc = run(None, 16, nh * hd, T, 4, 4, 2, nh, kv, 16, 0.1, window, T, L, 16, n, None)
                            assert rc == -1 and "null ctx" in _lib.last_error(), (T, L, window, _lib.last_error())


class HostDevice:
    """Device memory as host byte arrays."""
    handle = None

    def __init__(self):
        self.mem = {}
        self.next = 4096

    def malloc(self, n):
        p, self.next = self.next, self.next + (n + 255) // 256 * 256
        self.mem[p] = np.zeros(n, np.uint8)
        return p

    def free(self, p):
        del self.mem[p]

    def _at(self, p):
        base = max(b for b in self.mem if b <= p)
        return self.mem[base][p - base:]

    def h2d(self, p, a):
        a = np.ascontiguousarray(a)
        self._at(p)[:a.nbytes] = a.reshape(-1).view(np.uint8)

    def d2h(self, a, p):
        a.reshape(-1).view(np.uint8)[:] = self._at(p)[:a.nbytes]
        return a

    def fill(self, p, value, n):
        self._at(p)[:n] = value

    def sync(self):
        pass


def test_page_account():
    dev = HostDevice()
    c = dr.PagedKVCache(2, n_pages=6, page=16, nkv=2, hd=8, max_seqs=3, max_pages=4, kv_dtype=LT_KV_F32, dev=dev)
    c.reserve(0, 17)
    c.reserve(1, 16)
    c.reserve(0, 20)                          # no new page
    c.reserve(0, 33)
    assert c.pages == [[0, 1, 3], [2], []]
    t = c.table.to_host()
    assert t.tolist() == [[0, 1, 3, -1], [2, -1, -1, -1], [-1] * 4]
    with pytest.raises(ValueError, match="at most 4"):
        c.reserve(1, 65)
    with pytest.raises(ValueError, match="2 free"):
        c.reserve(2, 48)
    assert c.pages[2] == [] and c.table.to_host()[2].tolist() == [-1] * 4
    c.set_lengths([33, 5, 0])
    c.release(0)
    assert c.lengths() == [0, 5, 0] and len(c.free_pages) == 5
    c.reserve(2, 48)
    assert len(set(c.pages[2] + c.pages[1])) == 4 and 2 not in c.pages[2]
    assert c.layers[0].desc.page == 16 and c.layers[0].desc.table == c.layers[1].desc.table
    c.free()
    assert not dev.mem


def test_descriptor_refusals():
    dev = HostDevice()
    k = dr.DevTensor.empty((4, 2, 16, 8), np.float32, dev)
    t = dr.DevTensor.zeros((1, 4), np.int32, dev)
    dr.PagedKV(k, k, t, LT_KV_F32)
    with pytest.raises(ValueError):
        dr.PagedKV(k, k, t, LT_KV_F16)
    with pytest.raises(ValueError):
        dr.PagedKV(k, k.view(0, (4, 2, 8, 16)), t, LT_KV_F32)
    with pytest.raises(ValueError):
        dr.PagedKV(k, k, t.view(0, (4,)), LT_KV_F32)
    with pytest.raises(ValueError):
        dr.PagedKVCache(1, 4, 24, 2, 8, 1, 4, dev=dev)
    with pytest.raises(ValueError):
        dr.PagedKVCache(1, 4, 16, 2, 8, 0, 4, dev=dev)


def test_python_entries_check_shapes():
    """Sequences without a length or a table row, outputs that are too small: refused before the library is called."""
    dev = HostDevice()

    def t(*shape, dt=np.float32):
        return dr.DevTensor.empty(shape, dt, dev)

    kv = dr.PagedKV(t(4, 2, 16, 8), t(4, 2, 16, 8), dr.DevTensor.zeros((2, 4), np.int32, dev), LT_KV_F32)
    q, out, fr = t(6, 64), t(6, 32), t(4)
    start3, start4, lens = t(3, dt=np.int32), t(4, dt=np.int32), t(2, dt=np.int32)
    with pytest.raises(_lib.LtError, match="null ctx"):
        dr.attn_paged_into(q, start3, lens, kv, 4, 0.3, out)
    for args in ((q, start4, lens, kv, 4, 0.3, out), (q, start3, t(1, dt=np.int32), kv, 4, 0.3, out),
                 (q, start3, lens, kv, 4, 0.3, t(5, 32))):
        with pytest.raises(ValueError):
            dr.attn_paged_into(*args)
    with pytest.raises(_lib.LtError, match="null ctx"):
        dr.rope_append_paged_into(q, out, start3, lens, 4, fr, kv)
    for args in ((q, out, start4, lens, 4, fr, kv), (q, t(5, 32), start3, lens, 4, fr, kv), (q, out, start3, lens, 4, t(3), kv)):
        with pytest.raises(ValueError):
            dr.rope_append_paged_into(*args)
    n = dr.verify_drafts_workspace_size(6, 100, True)
    i32 = np.int32
    good = dict(logits=t(6, 100), toks=t(6, dt=i32), q_start=start3, u=t(6), params=t(64, dt=np.uint8), out_tok=t(6, dt=i32),
                n_out=t(2, dt=i32), ws=t(n, dt=np.uint8), draft_logits=t(6, 100), lens=lens)
    with pytest.raises(_lib.LtError, match="null ctx"):
        dr.verify_drafts_into(**good)
    for bad in (dict(toks=t(5, dt=i32)), dict(u=t(5)), dict(out_tok=t(5, dt=i32)), dict(n_out=t(1, dt=i32)),
                dict(params=t(63, dt=np.uint8)), dict(draft_logits=t(6, 99)), dict(lens=t(1, dt=i32))):
        with pytest.raises(ValueError):
            dr.verify_drafts_into(**{**good, **bad})


def test_page_account_takes_only_its_sequences():
    """A sequence number outside the cache would address device memory before or behind the table and the lengths."""
    c = dr.PagedKVCache(1, 4, 16, 2, 8, max_seqs=2, max_pages=2, kv_dtype=LT_KV_F32, dev=HostDevice())
    for b in (-1, 2):
        with pytest.raises(ValueError, match="cache of 2"):
            c.reserve(b, 1)
        with pytest.raises(ValueError, match="cache of 2"):
            c.release(b)
    assert c.pages == [[], []] and len(c.free_pages) == 4
