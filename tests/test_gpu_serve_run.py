"""The packed-batch operators as a server uses them: page plan, DeltaNet block and attention layer one after the other over
steps in which requests come, grow and end; captured into a graph; on streams of their own; over shared pages."""

import numpy as np
import pytest

import hiprt
import oracle
from oracle import serve

pytestmark = pytest.mark.gpu

# as in the tests of each operator: fp32 sums of operands that keep 22 bits and more
TOL = 1e-5
D, HD = 128, 256


def _say(*a):
    print(*a, flush=True)


class Server:
    """One DeltaNet block and one attention layer over B request places, T rows a step, on device buffers."""

    ACT = ("qkv", "ab", "z", "qg", "k", "v")

    def __init__(self, L, B=4, T=96, nkh=2, nvh=4, nq=4, nkv=2, npages=24, mb=6, nsplit=3, seed=0):
        self.L, self.B, self.T, self.nkh, self.nvh, self.nq, self.nkv = L, B, T, nkh, nvh, nq, nkv
        self.npages, self.mb, self.nsplit = npages, mb, nsplit
        r = np.random.default_rng(seed)
        n = lambda *s: r.standard_normal(s).astype(np.float32)  # noqa: E731
        self.C = (2 * nkh + nvh) * D
        self.w = dict(conv_w=0.3 * n(self.C, 4), dt_bias=0.5 * n(nvh), ssm_a=-np.exp(0.5 * n(nvh)), norm_w=1 + 0.1 * n(D),
                      wq=1 + 0.1 * n(HD), wk=1 + 0.1 * n(HD))
        z = lambda *s: np.zeros(s, np.int32)  # noqa: E731
        self.state = dict(past=z(B), nnew=z(B), done=z(B), free=r.permutation(npages).astype(np.int32),
                          top=np.array([npages], np.int32), table=z(B, mb) - 1, cu=z(B + 1), slot=z(T), seq=z(T),
                          S=np.zeros((B, nvh, D, D), np.float32), ring=np.zeros((B, 4, self.C), np.float32),
                          cache=r.integers(0, 256, (npages, nkv, serve.HEAD_BYTES)).astype(np.uint8))
        self.wb = L.attn_kv4_work_bytes(B, T, nq, nkv, nsplit), L.gdn_chunk_work_bytes(B, T, nkh, nvh)
        self.d = {k: hiprt.Buf.like(a) for k, a in {**self.w, **self.state, **self.inputs(0),
                  "out": np.zeros((T, nvh * D), np.float32), "og": np.zeros((T, nq, HD), np.float32),
                  "aw": np.full(self.wb[0], 255, np.uint8), "gw": np.full(self.wb[1], 255, np.uint8)}.items()}

    def inputs(self, seed):
        r = np.random.default_rng(seed)
        n = lambda *s: r.standard_normal((self.T, *s)).astype(np.float32)  # noqa: E731
        return dict(qkv=n(self.C), ab=n(2 * self.nvh), z=n(self.nvh * D), qg=n(self.nq, 2, HD), k=n(self.nkv, HD), v=n(self.nkv, HD))

    def put(self, **kw):
        for k, a in kw.items():
            self.d[k].upload(a)

    def get(self, *names):
        return [self.d[k].download() for k in names]

    def launch(self, stream=0):
        p = {k: b.ptr for k, b in self.d.items()}
        L, B, T = self.L, self.B, self.T
        L.page_plan_dev(B, T, self.mb, self.npages, p["past"], p["nnew"], p["free"], p["top"], p["top"], p["table"], p["cu"],
                        p["slot"], p["seq"], stream=stream)
        L.gdn_block_chunk_dev(B, T, self.nkh, self.nvh, 4, *(p[k] for k in ("cu", "past", "qkv", "conv_w", "ring", "ab", "dt_bias",
                              "ssm_a", "S", "z", "norm_w", "out", "gw")), self.wb[1], stream=stream)
        L.attn_kv4_dev(B, T, self.nq, self.nkv, self.mb, self.npages, *(p[k] for k in ("past", "cu", "table", "slot", "seq", "qg",
                       "k", "v", "wq", "wk", "cache")), self.nsplit, p["aw"], self.wb[0], p["og"], stream=stream)

    def release(self, done):
        self.put(done=np.array(done, np.int32))
        p = {k: b.ptr for k, b in self.d.items()}
        self.L.page_release_dev(self.B, self.mb, self.npages, p["done"], p["past"], p["free"], p["top"], p["table"])
        hiprt.sync()

    def advance(self):
        past, nnew = self.get("past", "nnew")
        self.put(past=past + nnew)


class Plain:
    """The same in 64 bits, from a server's state."""

    def __init__(self, s):
        self.s = s
        self.past, self.free, self.table = (s.state[k].copy() for k in ("past", "free", "table"))
        self.top, self.cache = int(s.state["top"][0]), s.state["cache"].copy()
        self.S, self.ring = s.state["S"].astype(np.float64), s.state["ring"].astype(np.float64)

    def step(self, nnew, x):
        s = self.s
        self.top, self.table, self.cu, self.slot, self.seq = serve.plan(self.past, nnew, s.T, s.mb, self.free, self.top, self.table)
        og = serve.attn_kv4(self.past, self.cu, self.table, self.slot, x["qg"], x["k"], x["v"], s.w["wq"], s.w["wk"], self.cache)
        out = np.zeros((self.cu[-1], s.nvh * D))
        for b in range(s.B):
            at, n, p = slice(self.cu[b], self.cu[b + 1]), self.cu[b + 1] - self.cu[b], int(self.past[b])
            if not n:
                continue
            conv, Sb = self.ring[b, [(p - i) % 4 for i in (3, 2, 1)]][None], self.S[b:b + 1].copy()
            a = [np.ascontiguousarray(x[k][at])[None] for k in ("qkv", "ab", "z")]
            out[at] = oracle.gdn_block(a[0], s.w["conv_w"], np.ascontiguousarray(conv), a[1], s.w["dt_bias"], s.w["ssm_a"], Sb, a[2],
                                       s.w["norm_w"], s.nkh, s.nvh)[0]
            self.S[b] = Sb[0]
            for i in range(1, min(3, n) + 1):
                self.ring[b, (p + n - i) % 4] = x["qkv"][self.cu[b + 1] - i]
        self.past = self.past + np.array(nnew, np.int32)
        return out, og

    def release(self, done):
        for b in np.flatnonzero(done):
            for i in range(serve.pages(self.past[b])):
                if self.table[b, i] >= 0:
                    self.free[self.top] = self.table[b, i]
                    self.top += 1
                self.table[b, i] = -1
            self.past[b] = 0


# (new tokens of the four places, places that end after the step)
STEPS = [([70, 5, 0, 1], []), ([1, 1, 40, 1], []), ([1, 0, 1, 1], [0, 3]), ([30, 1, 1, 63], []), ([1, 1, 1, 1], [1]),
         ([1, 90, 1, 2], [2]), ([0, 0, 0, 0], []), ([4, 4, 64, 4], [0, 1, 2, 3]), ([96, 0, 0, 0], [])]


def test_requests_come_grow_and_end(fnlib):
    _say("server run")
    s = Server(fnlib)
    ref = Plain(s)
    fnlib.dev_status()
    for i, (nnew, done) in enumerate(STEPS):
        _say("step", i, nnew)
        x = s.inputs(i)
        # a new request starts from an empty state
        for b in range(s.B):
            if ref.past[b] == 0:
                ref.S[b], ref.ring[b] = 0, 0
        S, ring = s.get("S", "ring")
        S[ref.past == 0], ring[ref.past == 0] = 0, 0
        s.put(nnew=np.array(nnew, np.int32), S=S, ring=ring, out=np.full((s.T, s.nvh * D), 7.5, np.float32),
              og=np.full((s.T, s.nq, HD), 7.5, np.float32), **x)
        s.launch()
        hiprt.sync()
        out, og = ref.step(nnew, x)
        n = ref.cu[-1]
        got = s.get("out", "og", "top", "table", "cu", "slot", "seq", "cache")
        for a, b in zip(got[2:7], (ref.top, ref.table, ref.cu, ref.slot, ref.seq)):
            assert np.array_equal(a if a.size > 1 else a[0], b)
        assert np.array_equal(got[7], ref.cache)
        assert (got[0][n:] == 7.5).all() and (got[1][n:] == 7.5).all()
        if n:
            e = oracle.relerr(got[0][:n], out), oracle.relerr(got[1][:n], og), oracle.relerr(s.get("S")[0], ref.S)
            _say("out, og, S", e)
            assert max(e) <= TOL
        s.advance()
        if done:
            flags = [int(b in done) for b in range(s.B)]
            s.release(flags)
            ref.release(flags)
            past, table, top = s.get("past", "table", "top")
            assert np.array_equal(past, ref.past) and np.array_equal(table, ref.table) and top[0] == ref.top
    assert fnlib.dev_status() == 0


def test_a_captured_step_replays(fnlib):
    """One graph of a step, replayed with other lengths, inputs and states, with eager steps and synchronizations of
    another server between the replays: every replay has the bits of an eager step."""
    _say("server graph")
    a, b = Server(fnlib, seed=1), Server(fnlib, seed=1)
    a.launch()  # (what is made at a first call is made before the capture)
    hiprt.sync()
    for k, v in a.state.items():
        a.put(**{k: v})
    st = hiprt.Stream()
    g = hiprt.Graph(st, lambda: a.launch(st.handle))
    names = ("out", "og", "S", "ring", "cache", "table", "cu", "slot", "seq", "top")
    try:
        for i, (nnew, done) in enumerate(STEPS[:6]):
            x = a.inputs(100 + i)
            for s in (a, b):
                s.put(nnew=np.array(nnew, np.int32), **x)
            hiprt.sync()
            g.launch()
            st.sync()
            b.launch()
            hiprt.sync()
            for k, p, q in zip(names, a.get(*names), b.get(*names)):
                assert np.array_equal(p, q), (i, k)
            for s in (a, b):
                s.advance()
                if done:
                    s.release([int(j in done) for j in range(s.B)])
    finally:
        g.destroy()
        st.destroy()


def test_two_servers_at_once(fnlib):
    """Two steps on two streams, each with its own buffers and workspaces, give the bits that each gives alone."""
    _say("two streams")
    pair, alone = [Server(fnlib, seed=s) for s in (5, 6)], [Server(fnlib, seed=s) for s in (5, 6)]
    streams = [hiprt.Stream() for _ in pair]
    names = ("out", "og", "S", "cache")
    try:
        for i, (nnew, _) in enumerate(STEPS[:2]):
            for j in range(2):
                for s in (pair[j], alone[j]):
                    s.put(nnew=np.array(nnew[::1 - 2 * j], np.int32), **s.inputs(10 * i + j))
            hiprt.sync()
            for s, t in zip(pair, streams):
                s.launch(t.handle)
            for t in streams:
                t.sync()
            for s, r in zip(pair, alone):
                r.launch()
                hiprt.sync()
                for k, p, q in zip(names, s.get(*names), r.get(*names)):
                    assert np.array_equal(p, q), k
                s.advance(), r.advance()
    finally:
        for t in streams:
            t.destroy()


def _attn(L, nsplit, past, cu, table, slot, seq, qg, k, v, wq, wk, cache, **kw):
    T, nq, nkv = qg.shape[0], qg.shape[1], k.shape[1]
    d = [hiprt.Buf.like(np.ascontiguousarray(a, dtype=a.dtype if a.dtype in (np.float32, np.uint8) else np.int32))
         for a in (np.asarray(past), np.asarray(cu), table, np.asarray(slot), np.asarray(seq), qg, k, v, wq, wk, cache)]
    og = hiprt.Buf.like(np.full((T, nq, HD), 7.5, np.float32))
    nsplit = nsplit or L.attn_kv4_nsplit(len(past), T, nq, nkv, table.shape[1] * 64)
    wb = L.attn_kv4_work_bytes(len(past), T, nq, nkv, nsplit)
    w = hiprt.Buf.like(np.full(wb, 255, np.uint8))
    L.attn_kv4_dev(len(past), T, nq, nkv, table.shape[1], cache.shape[0], *(b.ptr for b in d), nsplit, w.ptr, wb, og.ptr, **kw)
    hiprt.sync()
    return og.download(), d[10].download()


def _batch(past, nnew, nq, nkv, T, seed):
    """A batch on a full page table of its own, tokens planned by the plain form."""
    r = np.random.default_rng(seed)
    n = lambda *s: r.standard_normal(s).astype(np.float32)  # noqa: E731
    mb = max(serve.pages(p + m) for p, m in zip(past, nnew))
    npages = mb * len(past)
    full = r.permutation(npages).reshape(len(past), mb)
    cache = r.integers(0, 256, (npages, nkv, serve.HEAD_BYTES)).astype(np.uint8)
    for b, p in enumerate(past):
        for i in range(p):
            serve.store(cache, int(full[b, i // 64]) * 64 + i % 64, n(nkv, HD), n(nkv, HD))
    cu = np.concatenate([[0], np.cumsum(nnew)])
    seq = np.full(T, -1)
    slot = np.full(T, -1)
    for b, (p, m) in enumerate(zip(past, nnew)):
        for i in range(m):
            seq[cu[b] + i], slot[cu[b] + i] = b, full[b, (p + i) // 64] * 64 + (p + i) % 64
    return dict(past=past, cu=cu, table=full, slot=slot, seq=seq, qg=n(T, nq, 2, HD), k=n(T, nkv, HD), v=n(T, nkv, HD),
                wq=1 + 0.1 * n(HD), wk=1 + 0.1 * n(HD), cache=cache)


# lengths and heads at the borders of the kernel's choices: items of 8 or 32 query rows (up to 24 rows a request, and one
# more), one launch for a token's queries and keys or two (T times groups of four tasks, against two a CU)
@pytest.mark.parametrize("past,nnew,nq,nkv,pad", [
    ([40, 7], [3, 3], 8, 1, 0), ([40, 7], [4, 3], 8, 1, 0), ([40, 7], [3, 4], 8, 1, 1), ([200, 90], [24, 24], 1, 1, 0),
    ([200, 90], [25, 24], 1, 1, 0), ([0], [560], 3, 1, 0), ([0, 100], [300, 1], 16, 4, 0), ([5, 66], [129, 127], 20, 5, 3),
    ([130], [1], 64, 1, 0), ([63, 0], [2, 700], 2, 2, 9)])
def test_attn_at_the_borders_of_its_variants(fnlib, past, nnew, nq, nkv, pad):
    _say("kv4 borders", past, nnew, nq, nkv)
    T = sum(nnew) + pad
    c = _batch(past, nnew, nq, nkv, T, seed=T)
    ref = {k: np.array(v, copy=True) for k, v in c.items()}
    og, cache = _attn(fnlib, 0, **c)
    want = serve.attn_kv4(*(ref[k] for k in ("past", "cu", "table", "slot", "qg", "k", "v", "wq", "wk", "cache")))
    n = sum(nnew)
    assert np.array_equal(cache, ref["cache"]) and (og[n:] == 7.5).all()
    e = oracle.relerr(og[:n], want)
    _say("og", e)
    assert e <= TOL


@pytest.mark.parametrize("nnew", [1, 9])
def test_attn_requests_that_share_pages(fnlib, nnew):
    """Requests with a common prefix name its pages in both tables; each appends behind it in pages of its own."""
    _say("kv4 shared pages", nnew)
    c = _batch([128, 128], [nnew, nnew], 8, 2, 2 * nnew, seed=3)
    c["table"][1, :2] = c["table"][0, :2]
    ref = {k: np.array(v, copy=True) for k, v in c.items()}
    og, cache = _attn(fnlib, 0, **c)
    want = serve.attn_kv4(*(ref[k] for k in ("past", "cu", "table", "slot", "qg", "k", "v", "wq", "wk", "cache")))
    assert np.array_equal(cache, ref["cache"])
    assert oracle.relerr(og, want) <= TOL


def test_attn_rows_disowned_by_their_request(fnlib):
    """A row whose seq names no request, or one whose rows it does not lie in, is not cached and is reported; the rows of
    other requests are as without it."""
    import fn

    _say("kv4 bad seq")
    c = _batch([30, 40, 50], [1, 1, 1], 8, 2, 3, seed=4)
    ref = {k: np.array(v, copy=True) for k, v in c.items()}
    c["seq"][1] = 7
    ref["slot"][1] = -1
    fnlib.dev_status()
    og, cache = _attn(fnlib, 2, **c)
    assert fnlib.dev_status() == fn.STATUS_ROWS
    want = serve.attn_kv4(*(ref[k] for k in ("past", "cu", "table", "slot", "qg", "k", "v", "wq", "wk", "cache")))
    assert np.array_equal(cache, ref["cache"])
    assert oracle.relerr(og[[0, 2]], want[[0, 2]]) <= TOL


def test_attn_far_pages(fnlib):
    """Pages whose bytes lie beyond 2^32 in the cache are read and written where they are."""
    _say("kv4 far pages")
    nkv = 8
    npages = (1 << 32) // fnlib.kv4_page_bytes(nkv) + 40
    c = _batch([100], [2], 8, nkv, 2, seed=5)
    ref = {k: np.array(v, copy=True) for k, v in c.items()}
    want = serve.attn_kv4(*(ref[k] for k in ("past", "cu", "table", "slot", "qg", "k", "v", "wq", "wk", "cache")))
    small = c["cache"]
    pb = fnlib.kv4_page_bytes(nkv)
    far = npages - small.shape[0] + np.arange(small.shape[0])
    big = hiprt.Buf(npages * pb, np.uint8)
    hiprt.htod(big.ptr + int(far[0]) * pb, small)
    d = {k: hiprt.Buf.like(np.ascontiguousarray(c[k], dtype=np.float32 if np.asarray(c[k]).dtype == np.float32 else np.int32))
         for k in ("past", "cu", "seq", "qg", "k", "v", "wq", "wk")}
    d["table"] = hiprt.Buf.like(far[c["table"]].astype(np.int32))
    d["slot"] = hiprt.Buf.like((far[c["slot"] // 64] * 64 + c["slot"] % 64).astype(np.int32))
    wb = fnlib.attn_kv4_work_bytes(1, 2, 8, nkv, 2)
    w, og = hiprt.Buf(wb, np.uint8), hiprt.Buf.empty((2, 8, HD))
    fnlib.attn_kv4_dev(1, 2, 8, nkv, c["table"].shape[1], npages, *(d[k].ptr for k in ("past", "cu", "table", "slot", "seq", "qg", "k",
                       "v", "wq", "wk")), big.ptr, 2, w.ptr, wb, og.ptr)
    hiprt.sync()
    assert np.array_equal(hiprt.dtoh(big.ptr + int(far[0]) * pb, small.shape, np.uint8), ref["cache"])
    assert oracle.relerr(og.download(), want) <= TOL


# one column tile a scan workgroup or two (B nvh 8 workgroups against the CUs), over several chunks
@pytest.mark.parametrize("lens,nkh,nvh", [([300], 16, 32), ([300], 11, 33), ([130, 64, 200], 4, 12), ([190] * 9, 2, 4)])
def test_gdn_core_columns(fnlib, lens, nkh, nvh):
    _say("core columns", lens, nkh, nvh)
    r = np.random.default_rng(nvh)
    n = lambda *s: r.standard_normal(s).astype(np.float32)  # noqa: E731
    B, T = len(lens), sum(lens)
    unit = lambda x: x / np.linalg.norm(x, axis=-1, keepdims=True)  # noqa: E731
    a = dict(q=unit(n(T, nkh, D)), k=unit(n(T, nkh, D)), v=n(T, nvh, D), beta=(1 / (1 + np.exp(-n(T, nvh)))).astype(np.float32),
             g=(-np.log1p(np.exp(n(T, nvh)))).astype(np.float32))
    S = 0.1 * n(B, nvh, D, D)
    cu = np.concatenate([[0], np.cumsum(lens)]).astype(np.int32)
    d = {k: hiprt.Buf.like(v) for k, v in {"cu": cu, **a, "S": S, "o": np.zeros((T, nvh, D), np.float32)}.items()}
    wb = fnlib.gdn_chunk_work_bytes(B, T, nkh, nvh)
    w = hiprt.Buf.like(np.full(wb, 255, np.uint8))
    fnlib.gdn_core_chunk_dev(B, T, nkh, nvh, *(b.ptr for b in d.values()), w.ptr, wb)
    hiprt.sync()
    o, rS = np.zeros((T, nvh, D)), S.astype(np.float64)
    for b in range(B):
        x, Sb = slice(cu[b], cu[b + 1]), rS[b:b + 1].copy()
        o[x] = oracle.gdn_core(*(np.ascontiguousarray(a[k][x])[None] for k in ("q", "k", "v", "beta", "g")), Sb)[0]
        rS[b] = Sb[0]
    e = oracle.relerr(d["o"].download(), o), oracle.relerr(d["S"].download(), rS)
    _say("o, S", e)
    assert max(e) <= TOL


# more requests than a wave has lanes: a request is found in two steps, and items come in their own order
# (with 16 query heads a kv head in items of 32 rows, with 8 in items of 8)
@pytest.mark.parametrize("B,new,nsplit,nq", [(64, 4, 1, 16), (65, 4, 1, 16), (70, 5, 3, 16), (300, 4, 1, 16), (150, 1, 2, 8), (70, 4, 1, 8)])
def test_attn_many_requests(fnlib, B, new, nsplit, nq):
    _say("kv4 many", B, new, nq)
    r = np.random.default_rng(B)
    past, nnew = r.integers(0, 150, B).tolist(), [int(x) for x in r.integers(0 if new > 1 else 1, new + 1, B)]
    c = _batch(past, nnew, nq, 1, sum(nnew) + 2, seed=B)
    ref = {k: np.array(v, copy=True) for k, v in c.items()}
    og, cache = _attn(fnlib, nsplit, **c)
    want = serve.attn_kv4(*(ref[k] for k in ("past", "cu", "table", "slot", "qg", "k", "v", "wq", "wk", "cache")))
    n = sum(nnew)
    assert np.array_equal(cache, ref["cache"]) and (og[n:] == 7.5).all()
    e = oracle.relerr(og[:n], want)
    _say("og", e)
    assert e <= TOL


def test_gdn_core_many_requests(fnlib):
    _say("core many")
    r = np.random.default_rng(9)
    n = lambda *s: r.standard_normal(s).astype(np.float32)  # noqa: E731
    lens = r.integers(0, 80, 200)
    lens[:5] = 0
    B, T, nkh, nvh = len(lens), int(lens.sum()) + 3, 1, 2
    unit = lambda x: x / np.linalg.norm(x, axis=-1, keepdims=True)  # noqa: E731
    a = dict(q=unit(n(T, nkh, D)), k=unit(n(T, nkh, D)), v=n(T, nvh, D), beta=(1 / (1 + np.exp(-n(T, nvh)))).astype(np.float32),
             g=(-np.log1p(np.exp(n(T, nvh)))).astype(np.float32))
    S = 0.1 * n(B, nvh, D, D)
    cu = np.concatenate([[0], np.cumsum(lens)]).astype(np.int32)
    d = {k: hiprt.Buf.like(v) for k, v in {"cu": cu, **a, "S": S, "o": np.full((T, nvh, D), 7.5, np.float32)}.items()}
    wb = fnlib.gdn_chunk_work_bytes(B, T, nkh, nvh)
    w = hiprt.Buf.like(np.full(wb, 255, np.uint8))
    fnlib.gdn_core_chunk_dev(B, T, nkh, nvh, *(b.ptr for b in d.values()), w.ptr, wb)
    hiprt.sync()
    o, rS = np.zeros((cu[-1], nvh, D)), S.astype(np.float64)
    for b in np.flatnonzero(lens):
        x, Sb = slice(cu[b], cu[b + 1]), rS[b:b + 1].copy()
        o[x] = oracle.gdn_core(*(np.ascontiguousarray(a[k][x])[None] for k in ("q", "k", "v", "beta", "g")), Sb)[0]
        rS[b] = Sb[0]
    got, gS = d["o"].download(), d["S"].download()
    assert (got[cu[-1]:] == 7.5).all() and np.array_equal(gS[lens == 0], S[lens == 0])
    e = oracle.relerr(got[:cu[-1]], o), oracle.relerr(gS, rS)
    _say("o, S", e)
    assert max(e) <= TOL


def test_plan_and_release_of_the_most_requests(fnlib):
    """8000 requests in one call, and all their pages back."""
    _say("plan 8000")
    r = np.random.default_rng(8)
    B, mb = 8000, 4
    past = r.integers(0, 190, B).astype(np.int32)
    nnew = r.integers(0, 3, B).astype(np.int32)
    T = int(nnew.sum()) + 1
    have = (past + 63) // 64
    npages = int(have.sum()) + 400
    order = r.permutation(npages).astype(np.int32)
    table = np.full((B, mb), -1, np.int32)
    table[np.arange(mb)[None] < have[:, None]] = order[:have.sum()]
    free = np.full(npages, -1, np.int32)
    free[:400] = order[have.sum():]
    z = lambda *s: np.zeros(s, np.int32)  # noqa: E731
    d = {k: hiprt.Buf.like(a) for k, a in dict(past=past, nnew=nnew, free=free, top=np.array([400], np.int32), table=table, cu=z(B + 1),
                                               slot=z(T), seq=z(T), done=z(B) + 1).items()}
    fnlib.dev_status()
    fnlib.page_plan_dev(B, T, mb, npages, d["past"].ptr, d["nnew"].ptr, d["free"].ptr, d["top"].ptr, d["top"].ptr, d["table"].ptr,
                        d["cu"].ptr, d["slot"].ptr, d["seq"].ptr)
    hiprt.sync()
    ref = serve.plan(past, nnew, T, mb, free, 400, table)
    for got, want in zip(("top", "table", "cu", "slot", "seq"), ref):
        assert np.array_equal(d[got].download().reshape(np.shape(want)), want), got
    d["past"].upload(past + nnew)
    fnlib.page_release_dev(B, mb, npages, d["done"].ptr, d["past"].ptr, d["free"].ptr, d["top"].ptr, d["table"].ptr)
    hiprt.sync()
    assert fnlib.dev_status() == 0
    assert d["top"].download()[0] == npages and np.array_equal(np.sort(d["free"].download()), np.arange(npages))
    assert (d["table"].download() == -1).all() and not d["past"].download().any()


# one workgroup for all tokens or many, with the count that is left in a place of its own and in the place that is read, and
# requests whose past stays in the LDS or not
@pytest.mark.parametrize("B,T,in_place", [(3, 4096, False), (3, 4097, False), (3, 4097, True), (40, 9000, False), (40, 9000, True),
                                          (5000, 5003, False), (5001, 5003, False), (5001, 5003, True)])
def test_plan_variants(fnlib, B, T, in_place):
    _say("plan variants", B, T, in_place)
    r = np.random.default_rng(T + B)
    past = r.integers(0, 200, B).astype(np.int32)
    past[1] = -3
    nnew = np.bincount(r.integers(0, B, T - 2), minlength=B).astype(np.int32)
    want = (np.maximum(past, 0) + nnew + 63) // 64
    mb = int(want.max()) - 1 if B == 40 else int(want.max())    # (of 40 requests some have tokens past the table)
    have = np.minimum((np.maximum(past, 0) + 63) // 64, mb)
    npages = int(have.sum()) + int((want - have).sum()) - (5 if B == 40 else 0)    # (and some pages are missing)
    order = r.permutation(npages).astype(np.int32)
    table = np.full((B, mb), -1, np.int32)
    table[np.arange(mb)[None] < have[:, None]] = order[:have.sum()]
    top = npages - int(have.sum())
    free = np.full(npages, -1, np.int32)
    free[:top] = order[have.sum():]
    z = lambda *s: np.zeros(s, np.int32) - 9  # noqa: E731
    d = {k: hiprt.Buf.like(a) for k, a in dict(past=past, nnew=nnew, free=free, top=np.array([top], np.int32), left=z(1), table=table,
                                               cu=z(B + 1), slot=z(T), seq=z(T)).items()}
    left = d["top"] if in_place else d["left"]
    fnlib.dev_status()
    fnlib.page_plan_dev(B, T, mb, npages, d["past"].ptr, d["nnew"].ptr, d["free"].ptr, d["top"].ptr, left.ptr, d["table"].ptr,
                        d["cu"].ptr, d["slot"].ptr, d["seq"].ptr)
    hiprt.sync()
    fnlib.dev_status()
    ref = serve.plan(past, nnew, T, mb, free, top, table)
    for got, want in zip((left, d["table"], d["cu"], d["slot"], d["seq"]), ref):
        assert np.array_equal(got.download().reshape(np.shape(want)), want)


@pytest.mark.parametrize("lens,nkh,nvh", [([40, 63, 64, 1, 17] * 60, 2, 4), ([1500], 16, 32), ([300] * 6, 16, 48)])
def test_gdn_core_repeats(fnlib, lens, nkh, nvh):
    """Many workgroups a CU, twelve times: the same bits whatever the workspace held."""
    _say("core repeats", len(lens), nkh, nvh)
    r = np.random.default_rng(17)
    n = lambda *s: r.standard_normal(s).astype(np.float32)  # noqa: E731
    B, T = len(lens), sum(lens)
    unit = lambda x: x / np.linalg.norm(x, axis=-1, keepdims=True)  # noqa: E731
    a = dict(q=unit(n(T, nkh, D)), k=unit(n(T, nkh, D)), v=n(T, nvh, D), beta=(1 / (1 + np.exp(-n(T, nvh)))).astype(np.float32),
             g=(-np.log1p(np.exp(n(T, nvh)))).astype(np.float32))
    S = 0.1 * n(B, nvh, D, D)
    cu = np.concatenate([[0], np.cumsum(lens)]).astype(np.int32)
    d = {k: hiprt.Buf.like(v) for k, v in {"cu": cu, **a, "S": S, "o": np.zeros((T, nvh, D), np.float32)}.items()}
    wb = fnlib.gdn_chunk_work_bytes(B, T, nkh, nvh)
    w = hiprt.Buf(wb, np.uint8)
    first = None
    for i in range(12):
        if i % 4 == 0:
            w.upload(np.full(wb, (255, 0, 60)[i // 4], np.uint8))
        d["S"].upload(S)
        fnlib.gdn_core_chunk_dev(B, T, nkh, nvh, *(b.ptr for b in d.values()), w.ptr, wb)
        hiprt.sync()
        got = d["o"].download(), d["S"].download()
        first = first or got
        assert np.isfinite(got[0]).all() and all(np.array_equal(x, y) for x, y in zip(got, first)), i


@pytest.mark.parametrize("past,nnew,nq,nkv", [([100, 900, 0, 33] * 10, [40, 3, 70, 1] * 10, 16, 2), ([500] * 40, [1] * 40, 16, 2),
                                              ([0], [700], 24, 2)])
def test_attn_repeats(fnlib, past, nnew, nq, nkv):
    """The same for the attention: the same bits of outputs and cache in every call."""
    _say("kv4 repeats", len(past), nq, nkv)
    c = _batch(past, nnew, nq, nkv, sum(nnew), seed=21)
    first = None
    for i in range(8):
        got = _attn(fnlib, 1 + i % 2 * 2 if len(past) == 1 else 2, **c)
        if len(past) == 1 and i % 2:    # another split: within rounding
            assert oracle.relerr(got[0], first[0]) <= TOL and np.array_equal(got[1], first[1])
            continue
        first = first or got
        assert np.isfinite(got[0]).all() and all(np.array_equal(x, y) for x, y in zip(got, first)), i
