"""GPU checks at the edges of the packed-batch operators: values that are not finite or hardly so, batches that are a part of
a larger one, and what the status word says."""

import numpy as np
import pytest

import fn
import hiprt
import oracle
from oracle import serve
from test_gpu_gdn_chunk import Block, Core
from test_gpu_serve import TOL, Batch, _run, _say

pytestmark = pytest.mark.gpu

# arguments of a gate: not finite, near the ends of fp32, around the place where e^-x leaves fp32 (88.72), ordinary
GATES = np.array([np.nan, np.inf, -np.inf, 3e38, -3e38, 2.4e38, -2.4e38, 1e38, -1e38, 1e5, -1e5, 104, -104, 89, -89, 88.73, -88.73,
                  88.7228, -88.7228, 88, -88, 87, -87, 20, -20, 1, -1, 0, -0.0], np.float32)


def _sigmoid(x):
    with np.errstate(over="ignore"):
        return 1.0 / (1.0 + np.exp(-np.asarray(x, np.float64)))


def _same(got, value, gate, what):
    """NaN where value * gate is, infinities alike, and within 1e-5 of it.  A gate below 2^-126 (a denormal of fp32) may be
    taken for 0, which moves the product by at most 2^-126 |value|; a product below 2^-126 may be too."""
    with np.errstate(invalid="ignore"):
        want = np.asarray(value, np.float64) * gate
    with np.errstate(over="ignore"):
        held = want.astype(np.float32)
    assert np.array_equal(np.isnan(got), np.isnan(held)), what
    inf = np.isinf(held)
    assert np.array_equal(got[inf], held[inf]), what
    f = np.isfinite(held)
    bad = np.abs(got[f] - want[f]) > TOL * np.abs(want[f]) + 2.0 ** -126 * (1.0 + np.abs(value[f]))
    assert not bad.any(), (what, got[f][bad][:5], want[f][bad][:5])


# an item of 8 rows and of 32, each with its keys in one split (the walk applies the gate) and in several (the join does)
@pytest.mark.parametrize("past,nnew", [([70, 3], [1, 1]), ([40, 0], [20, 9])])
@pytest.mark.parametrize("nsplit", [1, 3])
def test_attn_gate_of_any_value(fnlib, past, nnew, nsplit):
    """The output is what it is under a gate of 1/2, times twice the sigmoid of the gate, whatever that is."""
    _say("kv4 gate", past, nnew, nsplit)
    c = Batch(past, nnew, nq=8, nkv=1, seed=31)
    c.qg[:, :, 1] = 0
    half, cache = _run(fnlib, c, nsplit)
    assert np.isfinite(half).all()
    gate = c.qg[:, :, 1]
    gate[...] = np.resize(GATES, gate.shape)
    og, again = _run(fnlib, c, nsplit)
    assert np.array_equal(cache, again)
    _same(og, 2.0 * half.astype(np.float64), _sigmoid(gate), "og")


@pytest.mark.parametrize("gate_act", [0, 1])
def test_block_gate_of_any_value(fnlib, gate_act):
    """The same for the block's z: the output under a gate of 1/2 times 2 sigmoid(z), or 2 z sigmoid(z)."""
    _say("block gate", gate_act)
    c = Block([0, 9], [70, 3], seed=32, gate_act=0)
    c.z[:] = 0
    half = c.run(fnlib)[0].astype(np.float64)
    assert np.isfinite(half).all()
    c.gate_act = gate_act
    c.z[...] = np.resize(GATES, c.z.shape)
    value = 2.0 * half * (c.z.astype(np.float64) if gate_act else 1.0)
    out = c.run(fnlib)[0]
    # (a product beyond fp32 on its way to a finite value may be infinite there)
    keep = (np.abs(value) < 1e37) | ~np.isfinite(value)
    _same(out[keep], value[keep], _sigmoid(c.z)[keep], "out")


@pytest.mark.parametrize("at", ["q", "k", "v"])
@pytest.mark.parametrize("x", [-100.0, -1e5, -1e38, -3e38])
def test_block_channels_far_below_zero(fnlib, at, x):
    """SiLU of a conv output far below zero is 0, and the head goes on as with a 0 there."""
    _say("block channel", at, x)
    c = Block([0, 9], [70, 3], seed=33)
    ch = {"q": 5, "k": c.nkh * 128 + 130, "v": 2 * c.nkh * 128 + 300}[at]
    c.conv_w[ch] = [0, 0, 0, 1]
    c.qkv[3::7, ch] = x
    out, S, _ = c.run(fnlib)
    ro, rS, _ = c.reference()
    e = oracle.relerr(out, ro), oracle.relerr(S, rS)
    _say("out, S", e)
    assert max(e) <= TOL


@pytest.mark.parametrize("x", [np.nan, np.inf, -np.inf])
def test_block_channels_not_finite(fnlib, x):
    """A value channel that is not finite leaves no finite output in its head from its token on, and reaches neither other
    heads nor other requests nor earlier chunks."""
    _say("block not finite", x)
    c = Block([0, 9], [140, 20], seed=34)
    ref, rS, _ = c.reference()
    head, t = 2, 100
    ch = 2 * c.nkh * 128 + head * 128 + 7
    c.conv_w[ch] = [0, 0, 0, 1]
    ref, rS, _ = c.reference()
    c.qkv[t, ch] = x
    out, S, _ = c.run(fnlib)
    out, ref = out.reshape(c.T, c.nvh, 128), ref.reshape(c.T, c.nvh, 128)
    assert not np.isfinite(out[t:140, head, 7]).any()
    keep = np.ones((c.T, c.nvh), bool)
    keep[64:140, head] = False
    assert oracle.relerr(out[keep], ref[keep]) <= TOL
    heads = [h for h in range(c.nvh) if h != head]
    assert oracle.relerr(S[0, heads], rS[0, heads]) <= TOL and oracle.relerr(S[1], rS[1]) <= TOL


# items of 8 and of 32 rows
ITEMS = [([300, 70], [1, 1]), ([200, 0], [3, 60])]


@pytest.mark.parametrize("past,nnew", ITEMS)
@pytest.mark.parametrize("e", [-99, -60, 60, 100, 125])
def test_attn_values_of_any_size(fnlib, past, nnew, e):
    """Values times 2^e, from the least that the format holds whole to its largest: the same codes, and the outputs times 2^e.
    (A product of the least value, 2^-101, and a probability is 2^-129 in the sums and rounds three times at 2^-150: 2^-19.4
    of it, within the bar.)"""
    _say("kv4 values", past, e)
    c = Batch(past, nnew, nq=8, nkv=1, seed=35)
    for b, p in enumerate(c.past):
        for i in range(p):
            s = int(c.full[b, i // 64]) * 64 + i % 64
            K, V = serve.load(c.cache, [s])
            serve.store(c.cache, s, K[0], np.ldexp(V[0], e))
    c.v = np.ldexp(c.v, e)
    ref = serve.attn_kv4(c.past, c.cu, c.full, c.slot, c.qg, c.k, c.v, c.wq, c.wk, c.cache.copy())
    for nsplit in (1, 3):
        og, _ = _run(fnlib, c, nsplit)
        r = oracle.relerr(np.ldexp(og.astype(np.float64), -e), np.ldexp(ref, -e))
        _say("og", nsplit, r)
        assert r <= TOL


@pytest.mark.parametrize("nnew", [1, 9])
def test_attn_largest_values_under_growing_scores(fnlib, nnew):
    """The largest value that the format holds in every place, under scores that grow by the most that a sum's reference lets
    pass (8.48 powers of two): the output is that value times the gate."""
    _say("kv4 largest", nnew)
    past, top = 5000, 6.0 * 2.0 ** 125
    c = Batch([past], [nnew], nq=8, nkv=1, seed=36)
    c.qg[:, :, 0], c.wq[:], c.wk[:] = 1, 0.98, 0.375      # queries of 0.98 in every dim; the new keys are 0.375
    c.k[:], c.v[:] = 1, top
    rows = {}
    for x in (0.0, 0.375):                                # 256 * 0.375 * 0.98 / 16 * log2(e) = 8.48
        one = np.zeros((1, 1, serve.HEAD_BYTES), np.uint8)
        for i in range(64):
            serve.store(one, i, np.full((1, 256), x), np.full((1, 256), top))
        rows[x] = one[0]
    for i in range(serve.pages(past)):
        c.cache[c.full[0, i]] = rows[0.0 if i < 8 else 0.375]
    for nsplit in (1, 3):
        og, _ = _run(fnlib, c, nsplit, nrot=0)
        want = top * _sigmoid(c.qg[:, :, 1])
        assert np.isfinite(og).all() and np.abs(og / want - 1).max() <= TOL


def test_block_of_a_part_of_a_batch(fnlib):
    """The call of the requests from the second on (cu does not start at 0): the first one's rows, state and ring are left as
    they were, the others have the bits of the call of all."""
    _say("block part")
    c = Block([4, 0, 9], [5, 70, 3], seed=37, pad=2)
    out, S, conv = c.run(fnlib)
    c.B, c.lens, c.cu, c.pos, c.S, c.conv = 2, c.lens[1:], c.cu[1:].copy(), c.pos[1:].copy(), c.S[1:].copy(), c.conv[1:].copy()
    part, pS, pconv = c.run(fnlib)
    assert (part[:5] == 7.5).all() and (part[78:] == 7.5).all()
    assert np.array_equal(part[5:78], out[5:78]) and np.array_equal(pS, S[1:]) and np.array_equal(pconv, conv[1:])


@pytest.mark.parametrize("nnew", [[2, 1, 1], [5, 40, 1]])
def test_attn_of_a_part_of_a_batch(fnlib, nnew):
    """The same for the attention: rows before cu[0] are no request's, nothing of them is written and nothing is wrong."""
    _say("kv4 part", nnew)
    c = Batch([20, 70, 33], nnew, nq=8, nkv=1, seed=38, pad=2)
    og, cache = _run(fnlib, c, 2)
    n, end = nnew[0], int(c.cu[-1])
    before = c.cache
    c.B, c.past, c.nnew, c.cu, c.full = 2, c.past[1:].copy(), c.nnew[1:].copy(), c.cu[1:].copy(), c.full[1:].copy()
    c.seq = np.maximum(c.seq - 1, -1)
    fnlib.dev_status()
    part, pcache = _run(fnlib, c, 2)
    assert fnlib.dev_status() == 0
    assert (part[:n] == 7.5).all() and (part[end:] == 7.5).all()
    ref = before.copy()
    want = serve.attn_kv4(c.past, c.cu - n, c.full, c.slot[n:], c.qg[n:], c.k[n:], c.v[n:], c.wq, c.wk, ref)
    assert np.array_equal(pcache, ref)
    assert oracle.relerr(part[n:end], want) <= TOL


# what is wrong with a plan, and the bits that say so
WRONG = {"nothing": 0, "pages": fn.STATUS_PAGE, "table": fn.STATUS_POS, "past": fn.STATUS_POS, "rows": fn.STATUS_ROWS,
         "count": fn.STATUS_ROWS, "pages and table": fn.STATUS_PAGE | fn.STATUS_POS, "lost page": fn.STATUS_PAGE}


# one workgroup for all tokens (up to 4096), many, and a second launch for the tokens (the count that is left in the place
# that is read); requests whose past stays in the LDS (up to 5000) or not
@pytest.mark.parametrize("wrong", list(WRONG))
@pytest.mark.parametrize("B,T,in_place", [(9, 600, False), (9, 600, True), (9, 4500, False), (9, 4500, True), (5001, 5200, False)])
def test_plan_says_what_is_wrong(fnlib, wrong, B, T, in_place):
    """Exactly the bits of what is wrong, in every way that a plan is launched, and the tables of the plain form beside."""
    _say("plan wrong", wrong, B, T, in_place)
    r = np.random.default_rng(B + T)
    past = r.integers(0, 200, B).astype(np.int32)
    nnew = np.bincount(r.integers(0, B, T - 3), minlength=B).astype(np.int32)
    past[2], nnew[2] = 100, 60
    rows = T = int(nnew.sum()) + 3
    want = (past + nnew + 63) // 64
    have = (past + 63) // 64
    mb = int(want.max())
    if "table" in wrong:
        mb -= 1
    if wrong == "past":
        past[2] = -4
    if wrong == "count":
        nnew[2] = -1
    if wrong == "rows":
        T = rows - 4
    need = int((np.minimum(want, mb) - np.minimum(have, mb)).clip(0).sum())
    npages = int(have.sum()) + need
    order = r.permutation(npages).astype(np.int32)
    have = np.minimum(have, mb)
    table = np.full((B, mb), -1, np.int32)
    table[np.arange(mb)[None] < have[:, None]] = order[:have.sum()]
    free = np.full(npages, -1, np.int32)
    free[:need] = order[have.sum():have.sum() + need]
    top = need - (2 if "pages" in wrong else 0)
    if wrong == "lost page":
        table[2, 1] = -1      # its past ends in this block, and new tokens go on in it
    z = lambda *n: np.zeros(n, np.int32) - 9  # noqa: E731
    d = {k: hiprt.Buf.like(a) for k, a in dict(past=past, nnew=nnew, free=free, top=np.array([top], np.int32), left=z(1), table=table,
                                               cu=z(B + 1), slot=z(T), seq=z(T)).items()}
    left = d["top"] if in_place else d["left"]
    fnlib.dev_status()
    fnlib.page_plan_dev(B, T, mb, npages, d["past"].ptr, d["nnew"].ptr, d["free"].ptr, d["top"].ptr, left.ptr, d["table"].ptr,
                        d["cu"].ptr, d["slot"].ptr, d["seq"].ptr)
    hiprt.sync()
    assert fnlib.dev_status() == WRONG[wrong]
    ref = serve.plan(past, nnew, T, mb, free, top, table)
    for got, x in zip((left, d["table"], d["cu"], d["slot"], d["seq"]), ref):
        assert np.array_equal(got.download().reshape(np.shape(x)), x)


@pytest.mark.parametrize("forget", [False, True])
@pytest.mark.parametrize("jump", [1e4, 1e6, 1e8, 1e12])
def test_core_values_that_fall(fnlib, jump, forget):
    """Values that fall within a chunk, with the ordinary decays and with one of 0 at the fall.  A column's operands are
    rounded at 2^-39 of its largest value or update; a row of M and of P sums 64 such with factors of 1 at most and 2^2.5
    in all for keys of random directions, one after the other: 2^-34 of the largest value.  What comes before the fall is at
    the bar."""
    _say("core fall", jump, forget)
    c = Core([64, 100], seed=40)
    fall = [32, 64 + 40]
    for a, b in ((0, fall[0]), (64, fall[1])):
        c.v[a:b] *= np.float32(jump)
    if forget:
        c.g[fall] = -np.inf
    o, S = c.run(fnlib)
    ro, rS = c.reference()
    top = np.abs(c.v).max()
    assert np.abs(o - ro).max() <= max(2.0 ** -34 * top, TOL * np.abs(ro).max())
    for a, b in ((0, fall[0]), (64, fall[1])):
        assert oracle.relerr(o[a:b], ro[a:b]) <= TOL
    for a, b in ((fall[0], 64), (fall[1], 128)):
        assert np.abs(o[a:b] - ro[a:b]).max() <= 2.0 ** -34 * top + TOL * np.abs(ro[a:b]).max()
    assert np.abs(S[0] - rS[0]).max() <= 2.0 ** -34 * top + TOL * np.abs(rS[0]).max()


def test_unpack_says_that_a_slot_is_outside(fnlib):
    """As packing does; a slot of -1 is no mistake.  Either way the row is left as it was."""
    _say("unpack outside")
    npages, n = 2, 4
    slot = np.array([5, -1, 127, -1], np.int32)
    cache = hiprt.Buf.like(np.full((npages, 1, serve.HEAD_BYTES), 127, np.uint8))
    k, v = (hiprt.Buf.like(np.full((n, 1, 256), 9.0, np.float32)) for _ in range(2))
    fnlib.dev_status()
    for bad, bits in ((-1, 0), (npages * 64, fn.STATUS_PAGE), (2 ** 31 - 1, fn.STATUS_PAGE)):
        slot[3] = bad
        d = hiprt.Buf.like(slot)
        fnlib.kv4_unpack_dev(n, 1, npages, d.ptr, cache.ptr, k.ptr, v.ptr)
        hiprt.sync()
        assert fnlib.dev_status() == bits, bad
        for x in (k.download(), v.download()):
            assert (x[[1, 3]] == 9.0).all() and (np.abs(x[[0, 2]]) == 6.0).all()    # (codes 7 and 15, scale 1)
