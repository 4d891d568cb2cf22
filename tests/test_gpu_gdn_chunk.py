"""GPU parity of the chunked delta rule over packed prompts against the float64 oracle, which goes token by token."""

import numpy as np
import pytest

import hiprt
import oracle

pytestmark = pytest.mark.gpu

# Products keep 22 to 24 bits of each operand and sum in fp32; a sum of 128 terms and the chunk's solve add a few
# roundings: the library's bar, which the one-token kernels are held to as well.
TOL = 1e-5
D = 128


def _say(*a):
    print(*a, flush=True)


class Core:
    def __init__(self, lens, nkh=2, nvh=4, head_map=0, seed=0, decay=1.0, pad=0):
        r = np.random.default_rng(seed)
        n = lambda *s: r.standard_normal(s).astype(np.float32)  # noqa: E731
        self.lens, self.nkh, self.nvh, self.head_map = lens, nkh, nvh, head_map
        self.cu = np.concatenate([[0], np.cumsum(lens)]).astype(np.int32)
        self.B, self.T = len(lens), int(self.cu[-1]) + pad
        unit = lambda x: x / np.linalg.norm(x, axis=-1, keepdims=True)  # noqa: E731
        self.q, self.k, self.v = unit(n(self.T, nkh, D)), unit(n(self.T, nkh, D)), n(self.T, nvh, D)
        self.beta = (1 / (1 + np.exp(-n(self.T, nvh)))).astype(np.float32)
        self.g = (-decay * np.log1p(np.exp(n(self.T, nvh)))).astype(np.float32)
        self.S = 0.1 * n(self.B, nvh, D, D)

    def run(self, L, stream=0):
        d = {x: hiprt.Buf.like(getattr(self, x)) for x in ("cu", "q", "k", "v", "beta", "g", "S")}
        o = hiprt.Buf.like(np.full((self.T, self.nvh, D), 7.5, np.float32))
        wb = L.gdn_chunk_work_bytes(self.B, self.T, self.nkh, self.nvh)
        w = hiprt.Buf.like(np.full(wb, 255, np.uint8))
        L.gdn_core_chunk_dev(self.B, self.T, self.nkh, self.nvh, *(d[x].ptr for x in ("cu", "q", "k", "v", "beta", "g", "S")),
                             o.ptr, w.ptr, wb, stream=stream, head_map=self.head_map)
        hiprt.sync()
        return o.download(), d["S"].download()

    def reference(self):
        S = self.S.astype(np.float64)
        o = np.zeros((int(self.cu[-1]), self.nvh, D))
        for b, n in enumerate(self.lens):
            if n:
                x = slice(self.cu[b], self.cu[b + 1])
                Sb = S[b:b + 1].copy()
                o[x] = oracle.gdn_core(*(np.ascontiguousarray(a[x])[None] for a in (self.q, self.k, self.v, self.beta, self.g)),
                                       Sb, head_map=self.head_map)[0]
                S[b] = Sb[0]
        return o, S

    def check(self, L, tol=TOL):
        o, S = self.run(L)
        ro, rS = self.reference()
        n = int(self.cu[-1])
        assert (o[n:] == 7.5).all()
        e = oracle.relerr(o[:n], ro), oracle.relerr(S, rS)
        _say("o, S", e)
        assert max(e) <= tol
        for b, m in enumerate(self.lens):
            if m == 0:
                assert np.array_equal(S[b], self.S[b])


@pytest.mark.parametrize("lens", [[1], [2], [15], [16], [17], [63], [64], [65], [128], [200], [1, 64, 0, 130, 5], [0, 0, 3], [1000]])
def test_core_lengths(fnlib, lens):
    _say("core", lens)
    Core(lens, seed=len(lens) + lens[0], pad=3).check(fnlib)


@pytest.mark.parametrize("nkh,nvh,head_map", [(1, 1, 0), (16, 32, 0), (16, 48, 1), (2, 6, 1), (3, 9, 0), (5, 5, 1)])
def test_core_heads(fnlib, nkh, nvh, head_map):
    _say("core heads", nkh, nvh, head_map)
    Core([70, 20], nkh, nvh, head_map, seed=nvh).check(fnlib)


@pytest.mark.parametrize("what", ["none", "strong", "underflow", "infinite", "mixed", "growing"])
def test_core_decays(fnlib, what):
    """Decays of 1, of almost 0, below fp32's range, of exactly 0, one strong decay among weak ones (whose sum must not
    cost the others their bits), and factors above 1."""
    _say("core decay", what)
    c = Core([150], seed=9)
    if what == "none":
        c.g[:] = 0
    elif what == "strong":
        c.g *= 20
    elif what == "underflow":
        c.g[:] = -150
    elif what == "infinite":
        c.g[10::17] = -np.inf
    elif what == "mixed":
        c.g *= 0.01
        c.g[5::40] = -190
    else:
        c.g[:] = 0.02
    c.check(fnlib)


@pytest.mark.parametrize("what", ["same keys", "beta 1", "beta 0", "zero keys", "keys", "values", "queries", "state", "rows"])
def test_core_values(fnlib, what):
    """Keys that repeat (the chunk's system is then the worst conditioned), betas of 1 and 0, and sizes far from 1: of the
    keys (the update's size goes with their square), values, queries and state, and from row to row."""
    _say("core values", what)
    c = Core([200, 30], seed=11)
    if what == "same keys":
        c.k[:] = c.k[0]
        c.beta[:] = 1
        c.g *= 0.01
    elif what == "beta 1":
        c.beta[:] = 1
    elif what == "beta 0":
        c.beta[:] = 0
    elif what == "zero keys":
        c.k[3::2] = 0
    elif what == "keys":
        c.k *= 0.01
    elif what == "values":
        c.v *= np.float32(1e12)
        c.S *= np.float32(1e12)
    elif what == "queries":
        c.q *= np.float32(1e-10)
    elif what == "state":
        c.S *= np.float32(1e-8)
    else:
        c.v *= np.exp(3 * np.random.default_rng(0).standard_normal((c.T, 1, 1))).astype(np.float32)
        c.q *= np.exp(5 * np.random.default_rng(1).standard_normal((c.T, 1, 1))).astype(np.float32)
    c.check(fnlib)


def test_core_long(fnlib):
    """A state carried over many chunks stays at the bar, with weak decays."""
    _say("core long")
    Core([5000], 1, 2, seed=13, decay=0.02).check(fnlib)


def test_core_neighbours(fnlib):
    """A NaN in one request reaches no other request and none of its own earlier chunks."""
    _say("core nan")
    c = Core([130, 100, 70], seed=15)
    ref, rS = c.reference()
    c.v[130 + 70, 1, 5] = np.nan
    o, S = c.run(fnlib)
    keep = np.ones(o.shape[:2], bool)
    keep[130 + 64:230, 1] = False
    assert np.isnan(o[130 + 70:230, 1, 5]).all()
    assert oracle.relerr(o[keep], ref[keep]) <= TOL
    assert oracle.relerr(S[[0, 2]], rS[[0, 2]]) <= TOL


class Block:
    def __init__(self, past, lens, nkh=2, nvh=4, head_map=0, gate_act=0, ring=4, seed=0, pad=0):
        r = np.random.default_rng(seed)
        n = lambda *s: r.standard_normal(s).astype(np.float32)  # noqa: E731
        self.lens, self.nkh, self.nvh, self.head_map, self.gate_act, self.ring = lens, nkh, nvh, head_map, gate_act, ring
        self.cu = np.concatenate([[0], np.cumsum(lens)]).astype(np.int32)
        self.B, self.T, C = len(lens), int(self.cu[-1]) + pad, (2 * nkh + nvh) * D
        self.pos = np.array(past, np.int32)
        self.qkv, self.conv_w, self.conv = n(self.T, C), 0.3 * n(C, 4), n(self.B, ring, C)
        self.ab, self.dt_bias, self.ssm_a = n(self.T, 2 * nvh), 0.5 * n(nvh), -np.exp(0.5 * n(nvh))
        self.S, self.z, self.norm_w = 0.1 * n(self.B, nvh, D, D), n(self.T, nvh * D), 1 + 0.1 * n(D)

    def run(self, L, stream=0):
        names = ("cu", "pos", "qkv", "conv_w", "conv", "ab", "dt_bias", "ssm_a", "S", "z", "norm_w")
        d = {x: hiprt.Buf.like(getattr(self, x)) for x in names}
        o = hiprt.Buf.like(np.full((self.T, self.nvh * D), 7.5, np.float32))
        wb = L.gdn_chunk_work_bytes(self.B, self.T, self.nkh, self.nvh)
        w = hiprt.Buf.like(np.full(wb, 255, np.uint8))
        L.gdn_block_chunk_dev(self.B, self.T, self.nkh, self.nvh, self.ring, *(d[x].ptr for x in names), o.ptr, w.ptr, wb,
                              stream=stream, head_map=self.head_map, gate_act=self.gate_act)
        hiprt.sync()
        return o.download(), d["S"].download(), d["conv"].download()

    def reference(self):
        S, ring = self.S.astype(np.float64), self.conv.astype(np.float64)
        o = np.zeros((int(self.cu[-1]), self.nvh * D))
        for b, n in enumerate(self.lens):
            if not n:
                continue
            x, p = slice(self.cu[b], self.cu[b + 1]), int(self.pos[b])
            conv, Sb = ring[b, [(p - d) % self.ring for d in (3, 2, 1)]][None], S[b:b + 1].copy()
            a = [np.ascontiguousarray(t[x])[None] for t in (self.qkv, self.ab, self.z)]
            o[x] = oracle.gdn_block(a[0], self.conv_w, np.ascontiguousarray(conv), a[1], self.dt_bias, self.ssm_a, Sb, a[2],
                                    self.norm_w, self.nkh, self.nvh, head_map=self.head_map, gate_act=self.gate_act)[0]
            S[b] = Sb[0]
            for d in range(1, min(3, n) + 1):
                ring[b, (p + n - d) % self.ring] = self.qkv[self.cu[b + 1] - d]
        return o, S, ring


@pytest.mark.parametrize("past,lens,kw", [([0], [1], {}), ([5], [2], {}), ([0, 7, 3], [70, 0, 3], {}), ([9], [130], dict(ring=16)),
                                          ([1000, 2], [64, 65], dict(head_map=1, gate_act=1)),
                                          ([3], [40], dict(nkh=16, nvh=48, gate_act=1)), ([0, 1], [200, 1], dict(nkh=16, nvh=32))])
def test_block(fnlib, past, lens, kw):
    _say("block", past, lens, kw)
    c = Block(past, lens, seed=len(lens), pad=2, **kw)
    o, S, conv = c.run(fnlib)
    ro, rS, rc = c.reference()
    n = int(c.cu[-1])
    assert (o[n:] == 7.5).all()
    assert np.array_equal(conv, rc.astype(np.float32))
    e = oracle.relerr(o[:n], ro), oracle.relerr(S, rS)
    _say("out, S", e)
    assert max(e) <= TOL


def test_block_continues(fnlib):
    """A prompt in two pieces, and then one token by fn_gdn_block_dev: what one call does."""
    _say("block in pieces")
    c = Block([0], [101], seed=21, ring=4)
    whole, S, conv = c.run(fnlib)
    pieces = []
    state = c.S, c.conv
    for a, b in ((0, 37), (37, 100)):
        p = Block([a], [b - a], seed=21)
        for x in ("qkv", "ab", "z"):
            setattr(p, x, np.ascontiguousarray(getattr(c, x)[a:b]))
        p.conv_w, p.dt_bias, p.ssm_a, p.norm_w, (p.S, p.conv) = c.conv_w, c.dt_bias, c.ssm_a, c.norm_w, state
        o, *state = p.run(fnlib)
        pieces.append(o)
    d = [hiprt.Buf.like(x) for x in (np.array([100], np.int32), c.qkv[100:], c.conv_w, state[1], c.ab[100:], c.dt_bias, c.ssm_a,
                                     state[0], c.z[100:], c.norm_w, np.zeros((1, c.nvh * D), np.float32))]
    fnlib.gdn_block_dev(1, c.nkh, c.nvh, 1, 4, *(x.ptr for x in d))
    hiprt.sync()
    pieces.append(d[10].download())
    assert oracle.relerr(np.concatenate(pieces), whole) <= TOL
    assert oracle.relerr(d[7].download(), S) <= TOL
    # the ring's fourth slot keeps what an earlier call left there
    live = [p % 4 for p in (98, 99, 100)]
    assert np.array_equal(d[3].download()[0, live], conv[0, live])
