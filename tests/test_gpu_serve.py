"""GPU parity of the packed-batch operators: page tables and the 4-bit paged cache with its attention, against plain
64-bit forms (oracle/serve.py)."""

import numpy as np
import pytest

import fn
import hiprt
import oracle
from oracle import serve

pytestmark = pytest.mark.gpu

# og: each step of the kernel is in fp32 or in parts that keep more than 24 bits (a query group 2^-24.9 of its largest
# value, probabilities 2^-25), V and K are exact.  A score of up to 2^8 rounds by 2^8 2^-24 a few times over, which moves
# a probability by as much: 2^-16 a row at the worst, far below in the norm over rows.  The library's bar is 1e-5.
TOL = 1e-5


def _say(*a):
    print(*a, flush=True)


def _i32(a):
    return np.ascontiguousarray(a, dtype=np.int32)


class Batch:
    """Requests with past[b] cached and nnew[b] new tokens, pages in random order, T >= the new tokens."""

    def __init__(self, past, nnew, nq=16, nkv=2, seed=0, spare=3, pad=0, max_blocks=None):
        r = np.random.default_rng(seed)
        self.past, self.nnew = _i32(past), _i32(nnew)
        self.B, self.nq, self.nkv = len(past), nq, nkv
        want = [serve.pages(p + n) for p, n in zip(past, nnew)]
        self.npages, self.mb = sum(want) + spare, max_blocks or max(want) + 1
        self.T = int(sum(nnew)) + pad
        order = _i32(r.permutation(self.npages))
        have = [serve.pages(p) for p in past]
        self.table = np.full((self.B, self.mb), -1, np.int32)
        at = 0
        for b, n in enumerate(have):
            self.table[b, :n] = order[at:at + n]
            at += n
        self.free = np.full(self.npages, -1, np.int32)
        self.free[:self.npages - at] = order[at:]
        self.top = self.npages - at
        _, self.full, cu, slot, seq = serve.plan(past, nnew, self.T, self.mb, self.free, self.top, self.table)
        self.cu, self.slot, self.seq = _i32(cu), _i32(slot), _i32(seq)
        n = lambda *s: r.standard_normal(s).astype(np.float32)  # noqa: E731
        self.qg, self.k, self.v = n(self.T, nq, 2, 256), n(self.T, nkv, 256), n(self.T, nkv, 256)
        self.wq, self.wk = 1 + 0.1 * n(256), 1 + 0.1 * n(256)
        self.cache = r.integers(0, 256, (self.npages, nkv, serve.HEAD_BYTES)).astype(np.uint8)  # unwritten rows: anything
        for b, p in enumerate(past):
            for i in range(p):
                serve.store(self.cache, int(self.full[b, i // 64]) * 64 + i % 64, n(nkv, 256), n(nkv, 256))


def _run(L, c, nsplit=0, stream=0, og=None, **kw):
    dev = {n: hiprt.Buf.like(getattr(c, n)) for n in ("past", "cu", "slot", "seq", "qg", "k", "v", "wq", "wk", "cache")}
    dev["table"] = hiprt.Buf.like(c.full)
    out = hiprt.Buf.like(np.full((c.T, c.nq, 256), 7.5, np.float32))
    nsplit = nsplit or L.attn_kv4_nsplit(c.B, c.T, c.nq, c.nkv, int((c.past + c.nnew).max()))
    wb = L.attn_kv4_work_bytes(c.B, c.T, c.nq, c.nkv, nsplit)
    work = hiprt.Buf.like(np.full(wb, 255, np.uint8))
    L.attn_kv4_dev(c.B, c.T, c.nq, c.nkv, c.mb, c.npages, *(dev[n].ptr for n in ("past", "cu", "table", "slot", "seq", "qg",
                   "k", "v", "wq", "wk", "cache")), nsplit, work.ptr, wb, out.ptr, stream=stream, **kw)
    hiprt.sync()
    return out.download(), dev["cache"].download()


def _check(L, c, nsplit=0, **kw):
    og, cache = _run(L, c, nsplit, **kw)
    ref_cache = c.cache.copy()
    ref = serve.attn_kv4(c.past, c.cu, c.full, c.slot, c.qg, c.k, c.v, c.wq, c.wk, ref_cache, **kw)
    n = int(c.cu[-1])
    assert np.array_equal(cache, ref_cache), int((cache != ref_cache).sum())
    assert (og[n:] == 7.5).all()
    e = oracle.relerr(og[:n], ref)
    _say("og", e)
    assert e <= TOL
    return og


@pytest.mark.parametrize("past,nnew", [([0], [1]), ([63], [1]), ([64], [1]), ([4095], [1]), ([5, 200, 0, 64], [1, 1, 1, 1]),
                                       ([100, 31], [4, 4]), ([0], [130]), ([0, 70, 300], [65, 1, 20]), ([7, 0, 9], [0, 3, 0])])
def test_attn_kv4_lengths(fnlib, past, nnew):
    _say("kv4", past, nnew)
    _check(fnlib, Batch(past, nnew, seed=len(past)))


@pytest.mark.parametrize("nq,nkv", [(1, 1), (8, 8), (4, 2), (24, 2), (12, 4), (15, 3), (48, 2), (20, 1)])
def test_attn_kv4_heads(fnlib, nq, nkv):
    _say("kv4 heads", nq, nkv)
    _check(fnlib, Batch([90, 3, 200], [1, 1, 1], nq, nkv, seed=nq))
    _check(fnlib, Batch([90, 3], [5, 70], nq, nkv, seed=nq))


@pytest.mark.parametrize("nsplit", [1, 2, 5, 40])
def test_attn_kv4_splits(fnlib, nsplit):
    """Any split of the keys gives the same within rounding; splits beyond the keys are empty."""
    _say("kv4 splits", nsplit)
    _check(fnlib, Batch([900, 10], [1, 1], seed=3), nsplit)
    _check(fnlib, Batch([400, 10], [9, 40], seed=4, pad=5), nsplit)


@pytest.mark.parametrize("nrot,theta,eps", [(0, 1e7, 1e-6), (64, 1e4, 1e-5), (128, 1e7, 1e-6), (50, 1e6, 0.0), (2, 1e7, 1e-6)])
def test_attn_kv4_rotation(fnlib, nrot, theta, eps):
    _say("kv4 rope", nrot)
    _check(fnlib, Batch([70, 8], [3, 1], seed=5), nrot=nrot, theta=theta, eps=eps)


def test_attn_kv4_far_position(fnlib):
    """A request at position 900,000 whose earlier blocks are not cached: angles of far positions, and blocks passed over."""
    _say("kv4 far")
    c = Batch([20, 70], [2, 1], seed=6, max_blocks=14100)
    c.past[1] = 900000
    c.full[1, :] = -1
    page = c.full[0, 0] + 1 if c.full[0, 0] + 1 < c.npages else 0
    c.full[1, 900000 // 64] = page
    c.slot[2] = page * 64 + 900000 % 64
    for i in range(64):
        serve.store(c.cache, int(page) * 64 + i, c.k[0] * (1 + i / 64), c.v[1])
    c.nnew[:] = [2, 1]
    og, _ = _run(fnlib, c, 3)
    assert fnlib.dev_status() & fn.STATUS_PAGE
    ref = serve.attn_kv4(c.past, c.cu, c.full, c.slot, c.qg, c.k, c.v, c.wq, c.wk, c.cache.copy())
    assert oracle.relerr(og, ref) <= TOL


@pytest.mark.parametrize("scale", [1e-30, 1e-3, 1e3, 1e30])
def test_attn_kv4_value_range(fnlib, scale):
    """Values far from 1: the scales are powers of two of the full fp32 range; scores in the hundreds."""
    _say("kv4 range", scale)
    c = Batch([130, 1], [2, 1], seed=7)
    c.v *= np.float32(scale)
    c.wq *= np.float32(30)
    for b, p in enumerate(c.past):
        for i in range(p):
            s = int(c.full[b, i // 64]) * 64 + i % 64
            K, V = serve.load(c.cache, [s])
            serve.store(c.cache, s, K[0], V[0] * scale)
    og, cache = _run(fnlib, c)
    rc = c.cache.copy()
    ref = serve.attn_kv4(c.past, c.cu, c.full, c.slot, c.qg, c.k, c.v, c.wq, c.wk, rc)
    assert np.array_equal(cache, rc)
    # scores reach 30 * 16: 480 2^-24 of a probability a rounding, eight of them
    assert oracle.relerr(og, ref) <= 8 * 480 * 2.0 ** -24


def test_attn_kv4_nonfinite(fnlib):
    """An infinity or NaN in a new key or value is stored as zeros, and the status word says so; in a query it makes
    its own output row NaN and no other."""
    _say("kv4 nonfinite")
    c = Batch([70, 9, 33], [1, 20, 1], seed=8)
    c.v[0, 1, 40] = np.inf
    c.k[3, 0, 9] = np.nan
    c.v[5, 0, 255] = -np.inf
    c.qg[7, 3, 0, 100] = np.nan
    c.qg[9, 15, 0, 0] = np.inf
    fnlib.dev_status()
    og, cache = _run(fnlib, c)
    assert fnlib.dev_status() == fn.STATUS_VALUE
    rc = c.cache.copy()
    ref = serve.attn_kv4(c.past, c.cu, c.full, c.slot, c.qg, c.k, c.v, c.wq, c.wk, rc)
    assert np.array_equal(cache, rc)
    bad = np.zeros(og.shape[:2], bool)
    bad[7, 3] = bad[9, 15] = True
    assert np.isnan(og[bad]).all() and np.isfinite(og[~bad]).all()
    assert oracle.relerr(og[~bad], ref[~bad]) <= TOL


def test_attn_kv4_no_key(fnlib):
    """A request none of whose blocks is cached gets zeros; a negative past too; the others are as without them."""
    _say("kv4 no key")
    c = Batch([70, 9, 33], [1, 3, 1], seed=9)
    c.full[1, :] = -1
    c.slot[1:4] = -1
    c.past[2] = -5
    c.slot[4] = -1
    og, _ = _run(fnlib, c)
    assert fnlib.dev_status() & (fn.STATUS_PAGE | fn.STATUS_POS) == fn.STATUS_PAGE | fn.STATUS_POS
    ref = serve.attn_kv4(c.past, c.cu, c.full, c.slot, c.qg, c.k, c.v, c.wq, c.wk, c.cache.copy())
    assert (og[1:] == 0).all()
    assert oracle.relerr(og, ref) <= TOL


def test_kv4_rows(fnlib):
    """Rows in and out of the cache: every byte of the layout, ties, borders, zeros, and slots passed over."""
    _say("kv4 rows")
    r = np.random.default_rng(1)
    n, nkv, npages = 150, 3, 4
    slot = _i32(r.permutation(npages * 64)[:n])
    slot[5], slot[9] = -1, npages * 64 + 3
    k, v = (r.standard_normal((n, nkv, 256)).astype(np.float32) for _ in range(2))
    k[0, 0, :32] = np.repeat([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0], 4)  # ties
    k[0, 1, :32] = np.linspace(-7, 7, 32)
    k[1, 0, :32] = [7.0] + [1.0] * 31
    k[1, 0, 32:64] = [np.nextafter(np.float32(7.0), np.float32(8))] + [1.0] * 31
    k[2, 0], k[2, 1], k[2, 2] = 0.0, 1e-38, 3e38
    v[3, 0, :64] = 2.0 ** -np.arange(64)
    v[4, 2, 77] = np.nan
    cache = r.integers(0, 256, (npages, nkv, serve.HEAD_BYTES)).astype(np.uint8)
    assert fnlib.kv4_page_bytes(nkv) == nkv * serve.HEAD_BYTES
    d = [hiprt.Buf.like(a) for a in (slot, k, v, cache)]
    fnlib.dev_status()
    fnlib.kv4_pack_dev(n, nkv, npages, *(b.ptr for b in d))
    hiprt.sync()
    assert fnlib.dev_status() == fn.STATUS_PAGE | fn.STATUS_VALUE
    ok = (slot >= 0) & (slot < npages * 64)
    for i in np.flatnonzero(ok):
        serve.store(cache, int(slot[i]), k[i], v[i])
    assert np.array_equal(d[3].download(), cache)
    out = [hiprt.Buf.like(np.full(k.shape, 9.0, np.float32)) for _ in range(2)]
    fnlib.kv4_unpack_dev(n, nkv, npages, d[0].ptr, d[3].ptr, out[0].ptr, out[1].ptr)
    hiprt.sync()
    K, V = serve.load(cache, slot[ok])
    for got, ref, x in zip(out, (K, V), (k, v)):
        got = got.download()
        assert np.array_equal(got[ok], ref.astype(np.float32)) and (got[~ok] == 9.0).all()
        # in scale units the largest value of a group lies in (3.5, 7] and a value up to 4 is off by at most 1/2, which is
        # 1/7 of 3.5; one above 4 by at most 1 and only at 5 by 1: at most 1/5 of the largest value
        x = x[ok].reshape(-1, 32)
        x, got = x[np.isfinite(x).all(1)], got[ok].reshape(-1, 32)[np.isfinite(x).all(1)]
        big = np.abs(x).max(1)
        assert (np.abs(got - x).max(1) <= big / 4.999)[big > 1e-29].all()


def _plan(L, c, nnew=None, T=None, in_place=False):
    T = T or c.T
    dev = {n: hiprt.Buf.like(a) for n, a in dict(past=c.past, nnew=_i32(c.nnew if nnew is None else nnew), free=c.free,
           top=_i32([c.top]), left=_i32([-9]), table=c.table, cu=_i32([-9] * (c.B + 1)), slot=_i32([-9] * T),
           seq=_i32([-9] * T)).items()}
    left = dev["top"] if in_place else dev["left"]
    L.page_plan_dev(c.B, T, c.mb, c.npages, *(dev[n].ptr for n in ("past", "nnew", "free", "top")), left.ptr,
                    *(dev[n].ptr for n in ("table", "cu", "slot", "seq")))
    hiprt.sync()
    return int(left.download()[0]), *(dev[n].download() for n in ("table", "cu", "slot", "seq")), dev


def _lens(past, nnew, **kw):
    """Batch's tables without its rows; lengths that do not fit are allowed."""
    c = Batch.__new__(Batch)
    r = np.random.default_rng(0)
    c.past, c.nnew, c.B = _i32(past), _i32(nnew), len(past)
    want = [serve.pages(max(p, 0) + max(n, 0)) for p, n in zip(past, nnew)]
    c.npages, c.mb = sum(want) + kw.get("spare", 3), kw.get("max_blocks") or max(want) + 1
    c.T = max(1, int(sum(max(n, 0) for n in nnew)) + kw.get("pad", 0))
    order = _i32(r.permutation(c.npages))
    c.table = np.full((c.B, c.mb), -1, np.int32)
    at = 0
    for b, p in enumerate(past):
        n = min(serve.pages(max(p, 0)), c.mb)
        c.table[b, :n] = order[at:at + n]
        at += n
    c.free = np.full(c.npages, -1, np.int32)
    c.free[:c.npages - at] = order[at:]
    c.top = c.npages - at
    return c


@pytest.mark.parametrize("past,nnew", [([0], [1]), ([0], [64]), ([64], [1]), ([63, 64, 65, 0], [1, 1, 1, 0]), ([10], [5000]),
                                       (list(range(0, 3000, 10)), [1] * 300), ([0] * 1500, [3] * 1500),
                                       ([5] * 40, [130] * 40)])
def test_page_plan(fnlib, past, nnew):
    _say("plan", len(past), sum(nnew))
    c = _lens(past, nnew, pad=7)
    fnlib.dev_status()
    for in_place in (False, True):
        left, table, cu, slot, seq, _ = _plan(fnlib, c, in_place=in_place)
        r = serve.plan(past, nnew, c.T, c.mb, c.free, c.top, c.table)
        assert left == r[0]
        for got, ref in zip((table, cu, slot, seq), r[1:]):
            assert np.array_equal(got, ref)
    assert fnlib.dev_status() == 0


@pytest.mark.parametrize("what", ["pages", "blocks", "rows", "counts"])
def test_page_plan_misuse(fnlib, what):
    """Too few pages, blocks past the table, more tokens than rows, negative counts: in bounds, and recorded."""
    _say("plan misuse", what)
    past, nnew, bit, T = [10, 100, 0], [100, 70, 200], fn.STATUS_PAGE, None
    kw = {}
    if what == "blocks":
        kw, bit = dict(max_blocks=2), fn.STATUS_POS
    if what == "counts":
        past, nnew, bit = [10, -100, 0], [100, 70, -200], fn.STATUS_ROWS | fn.STATUS_POS
    c = _lens(past, nnew, **kw)
    if what == "pages":
        c.top = 3
    if what == "rows":
        T, bit = 150, fn.STATUS_ROWS
    fnlib.dev_status()
    left, table, cu, slot, seq, _ = _plan(fnlib, c, T=T)
    assert fnlib.dev_status() == bit
    r = serve.plan(past, nnew, T or c.T, c.mb, c.free, c.top, c.table)
    assert left == r[0]
    for got, ref in zip((table, cu, slot, seq), r[1:]):
        assert np.array_equal(got, ref)


def test_page_release(fnlib):
    """Pages of ended requests come back in order, blocks without a page give none, and the next plan uses them."""
    _say("release")
    c = _lens([130, 64, 0, 500, 1], [1] * 5)
    c.table[3, 4] = -1
    done = _i32([1, 0, 1, 7, 0])
    d = {n: hiprt.Buf.like(a) for n, a in dict(done=done, past=c.past, free=c.free, top=_i32([c.top]), table=c.table).items()}
    fnlib.page_release_dev(c.B, c.mb, c.npages, *(d[n].ptr for n in ("done", "past", "free", "top", "table")))
    hiprt.sync()
    back = [int(p) for b in (0, 3) for p in c.table[b, :serve.pages(c.past[b])] if p >= 0]
    assert d["top"].download()[0] == c.top + len(back)
    free = d["free"].download()
    assert free[c.top:c.top + len(back)].tolist() == back and np.array_equal(free[:c.top], c.free[:c.top])
    assert d["past"].download().tolist() == [0, 64, 0, 0, 1]
    t = d["table"].download()
    assert (t[0, :3] == -1).all() and (t[3, :8] == -1).all() and np.array_equal(t[[1, 4]], c.table[[1, 4]])
    assert fnlib.dev_status() == 0
