"""CPU checks of the packed-batch operators: the plain 64-bit forms against direct definitions, and what the entry points
refuse before any device work."""

import numpy as np
import pytest

import fn
from oracle import serve

P = 4096  # an address that is 16-byte aligned; every call here is refused before it is read
BIG = 1 << 40

PLAN = dict(B=2, T=8, max_blocks=4, npages=16, past=P, nnew=P, free=P, top=P, left=P, table=P, cu=P, slot=P, seq=P)
RELEASE = dict(B=2, max_blocks=4, npages=16, done=P, past=P, free=P, top=P, table=P)
ROWS = dict(n=3, nkv=2, npages=4, slot=P, k=P, v=P, cache=P)
ATTN = dict(B=2, T=8, nq=16, nkv=2, max_blocks=4, npages=16, past=P, cu=P, table=P, slot=P, seq=P, qg=P, k=P, v=P, wq=P,
            wk=P, cache=P, nsplit=2, work=P, work_bytes=BIG, og=P)
CORE = dict(B=2, T=100, nkh=2, nvh=4, cu=P, q=P, k=P, v=P, beta=P, g=P, S=P, o=P, work=P, work_bytes=BIG)
BLOCK = dict(B=2, T=100, nkh=2, nvh=4, ring=4, cu=P, pos=P, qkv=P, conv_w=P, conv_ring=P, ab=P, dt_bias=P, ssm_a=P, S=P,
             z=P, norm_w=P, out=P, work=P, work_bytes=BIG)
CALLS = dict(page_plan_dev=PLAN, page_release_dev=RELEASE, kv4_pack_dev=ROWS, kv4_unpack_dev=ROWS, attn_kv4_dev=ATTN,
             gdn_core_chunk_dev=CORE, gdn_block_chunk_dev=BLOCK)
OPTIONS = ("hd", "nrot", "theta", "dk", "dv", "head_map", "gate_act")


def _refused(fnlib, call, match, **bad):
    args = dict(CALLS[call], **{k: v for k, v in bad.items() if k not in OPTIONS})
    with pytest.raises(RuntimeError, match=match):
        getattr(fnlib, call)(*args.values(), **{k: v for k, v in bad.items() if k in OPTIONS})


@pytest.mark.parametrize("call", list(CALLS))
def test_null_pointers_are_refused(fnlib, call):
    for name, value in CALLS[call].items():
        if value == P:
            _refused(fnlib, call, "null pointer", **{name: None})


@pytest.mark.parametrize("call,names", [("kv4_pack_dev", "k v cache"), ("kv4_unpack_dev", "k v cache"),
                                        ("attn_kv4_dev", "qg k v wq wk cache work og"), ("gdn_core_chunk_dev", "q k o work"),
                                        ("gdn_block_chunk_dev", "conv_w z norm_w out work")])
def test_unaligned_pointers_are_refused(fnlib, call, names):
    for name in names.split():
        for off in (4, 8):
            _refused(fnlib, call, "16-byte aligned", **{name: P + off})


@pytest.mark.parametrize("call,match,bad", [
    ("page_plan_dev", "B must be", dict(B=0)), ("page_plan_dev", "B must be", dict(B=8001)),
    ("page_plan_dev", "T must be", dict(T=0)), ("page_plan_dev", "T must be", dict(T=(1 << 30) + 1)),
    ("page_plan_dev", "max_blocks", dict(max_blocks=0)),
    ("page_plan_dev", "npages", dict(npages=0)), ("page_plan_dev", "npages", dict(npages=1 << 25)),
    ("page_release_dev", "B must be", dict(B=-1)), ("page_release_dev", "npages", dict(npages=1 << 25)),
    ("kv4_pack_dev", "n and nkv", dict(n=0)), ("kv4_pack_dev", "n and nkv", dict(nkv=0)),
    ("kv4_pack_dev", "nkv must be", dict(nkv=65536)), ("kv4_pack_dev", "head_dim 256", dict(hd=128)),
    ("kv4_unpack_dev", "npages", dict(npages=-1)), ("kv4_unpack_dev", "head_dim 256", dict(hd=64)),
    ("attn_kv4_dev", "must be >= 1", dict(B=0)), ("attn_kv4_dev", "must be >= 1", dict(T=0)),
    ("attn_kv4_dev", "must be >= 1", dict(nkv=0)), ("attn_kv4_dev", "multiple of nkv", dict(nq=5)),
    ("attn_kv4_dev", "head_dim 256", dict(hd=128)), ("attn_kv4_dev", "nrot", dict(nrot=63)),
    ("attn_kv4_dev", "nrot", dict(nrot=130)), ("attn_kv4_dev", "nrot", dict(nrot=-2)),
    ("attn_kv4_dev", "theta", dict(theta=0.5)), ("attn_kv4_dev", "theta", dict(theta=float("nan"))),
    ("attn_kv4_dev", "nsplit", dict(nsplit=0)), ("attn_kv4_dev", "nsplit", dict(nsplit=65536)),
    ("attn_kv4_dev", "max_blocks", dict(max_blocks=0)), ("attn_kv4_dev", "max_blocks", dict(max_blocks=(1 << 24) + 1)),
    ("attn_kv4_dev", "npages", dict(npages=1 << 25)), ("attn_kv4_dev", "too many query rows", dict(T=1 << 28)),
    ("attn_kv4_dev", "batch too large", dict(B=70000, T=70000)), ("attn_kv4_dev", "batch too large", dict(T=1 << 20)),
    ("gdn_core_chunk_dev", "must be >= 1", dict(B=0)), ("gdn_core_chunk_dev", "must be >= 1", dict(T=0)),
    ("gdn_core_chunk_dev", "dk = dv = 128", dict(dk=64)), ("gdn_core_chunk_dev", "dk = dv = 128", dict(dv=256)),
    ("gdn_core_chunk_dev", "multiple of nkh", dict(nvh=5)), ("gdn_core_chunk_dev", "head_map", dict(head_map=2)),
    ("gdn_core_chunk_dev", "<= 65535", dict(B=65536)), ("gdn_core_chunk_dev", "<= 32768", dict(nkh=1, nvh=32769)),
    ("gdn_block_chunk_dev", "gate_act", dict(gate_act=2)), ("gdn_block_chunk_dev", "ring", dict(ring=3)),
    ("gdn_block_chunk_dev", "ring", dict(ring=2)), ("gdn_block_chunk_dev", "ring", dict(ring=12)),
])
def test_bad_arguments_are_refused(fnlib, call, match, bad):
    _refused(fnlib, call, match, **bad)


@pytest.mark.parametrize("call,size", [("attn_kv4_dev", lambda L: L.attn_kv4_work_bytes(2, 8, 16, 2, 2)),
                                       ("gdn_core_chunk_dev", lambda L: L.gdn_chunk_work_bytes(2, 100, 2, 4)),
                                       ("gdn_block_chunk_dev", lambda L: L.gdn_chunk_work_bytes(2, 100, 2, 4))])
def test_small_workspaces_are_refused(fnlib, call, size):
    need = size(fnlib)
    assert need > 0
    for wb in (0, need - 1):
        _refused(fnlib, call, "workspace too small", work_bytes=wb)


def test_sizes(fnlib):
    """Sizes grow with every argument, and arguments that no call takes give 0 (splits: 1)."""
    L = fnlib
    assert L.kv4_page_bytes(2) == 2 * serve.HEAD_BYTES and L.kv4_page_bytes(0) == 0 and L.kv4_page_bytes(2, 128) == 0
    a = L.attn_kv4_work_bytes(4, 64, 16, 2, 4)
    assert 0 < a < L.attn_kv4_work_bytes(4, 128, 16, 2, 4) and a < L.attn_kv4_work_bytes(4, 64, 16, 2, 8)
    for bad in ((0, 1, 16, 2, 1), (1, 0, 16, 2, 1), (1, 1, 5, 2, 1), (1, 1, 16, 2, 0)):
        assert L.attn_kv4_work_bytes(*bad) == 0
    for bad in ((0, 1, 16, 2, 100), (1, 1, 5, 2, 100), (1, 1, 16, 2, 0), (1, 1, 16, 2, -7)):
        assert L.attn_kv4_nsplit(*bad) == 1
    g = L.gdn_chunk_work_bytes(1, 64, 2, 4)
    assert 0 < g < L.gdn_chunk_work_bytes(1, 128, 2, 4) and g < L.gdn_chunk_work_bytes(2, 64, 2, 4)
    assert L.gdn_chunk_work_bytes(1, 0, 2, 4) == 0
    assert fn.STATUS_PAGE == 4 and fn.STATUS_ROWS == 8 and fn.STATUS_VALUE == 16


def test_quantise_is_the_nearest_code():
    """Against every code under every scale: the scale is the least that leaves the largest value off by at most half a
    step, and each value gets the nearest level, a tie the even code."""
    r = np.random.default_rng(0)
    x = (r.standard_normal((200, 256)) * np.exp(4 * r.standard_normal((200, 1)))).astype(np.float32)
    x[0, :32] = 0
    x[1, :8] = [7, 3.5, 0.25, 0.75, 5, 2.5, 1.25, -1.75]
    x[1, 8:32] = 0
    x[2, :32] = np.nextafter(np.float32(7), np.float32(8))
    code, scale = serve.quantise(x)
    got = serve.values(code, scale)
    for i in range(200):
        for g in range(8):
            v = x[i, 32 * g:32 * g + 32].astype(np.float64)
            a = np.abs(v).max()
            e = -100
            while a > 7 * 2.0 ** e:      # half a step past the largest level, 6
                e += 1
            assert scale[i, g] == e + 127
            d = np.abs(np.abs(v)[:, None] - serve.LEVELS * 2.0 ** e)
            assert (np.abs(got[i, 32 * g:32 * g + 32] - v) == d.min(1)).all()
            tie = (d == d.min(1)[:, None]).sum(1) > 1
            assert (code[i, 32 * g:32 * g + 32][tie] % 2 == 0).all()


def test_layout_holds_every_value_once():
    kc, ks, vc, vs, sh = serve.offsets()
    for c in (kc, vc):
        assert len(np.unique(c * 2 + (sh > 0))) == c.size
    parts = [np.unique(o) for o in (kc, ks, vc, vs)]
    assert np.array_equal(np.sort(np.concatenate(parts)), np.arange(serve.HEAD_BYTES))
    r = np.random.default_rng(1)
    cache = np.zeros((2, 3, serve.HEAD_BYTES), np.uint8)
    k, v = r.standard_normal((2, 128, 3, 256))
    for s in range(128):
        serve.store(cache, s, k[s], v[s])
    K, V = serve.load(cache, np.arange(128))
    for got, x in ((K, k), (V, v)):
        assert np.array_equal(got, serve.values(*serve.quantise(x)))


@pytest.mark.parametrize("nrot", [0, 50, 128])
def test_attention_form_is_softmax(nrot):
    """The plain attention against a dense softmax over all tokens of one request."""
    r = np.random.default_rng(2)
    n, nq, nkv, past = 70, 4, 2, 30
    table = np.array([[1, 0]])
    cache = np.zeros((2, nkv, serve.HEAD_BYTES), np.uint8)
    old = r.standard_normal((2, past, nkv, 256))
    for i in range(past):
        serve.store(cache, int(table[0, 0]) * 64 + i, old[0, i], old[1, i])
    qg, k, v = r.standard_normal((n, nq, 2, 256)), r.standard_normal((n, nkv, 256)), r.standard_normal((n, nkv, 256))
    wq, wk = r.standard_normal(256), r.standard_normal(256)
    slot = np.array([table[0, p // 64] * 64 + p % 64 for p in range(past, past + n)])
    og = serve.attn_kv4([past], [0, n], table, slot, qg, k, v, wq, wk, cache, nrot=nrot, theta=1e4)

    pos = past + np.arange(n)
    q = serve.norm_rope(qg[:, :, 0], wq, pos, nrot, 1e4, 1e-6)
    K = np.concatenate([serve.values(*serve.quantise(old[0])), serve.values(*serve.quantise(serve.norm_rope(k, wk, pos, nrot, 1e4, 1e-6)))])
    V = np.concatenate([serve.values(*serve.quantise(old[1])), serve.values(*serve.quantise(v))])
    for h in range(nq):
        s = q[:, h] @ K[:, h // 2].T / 16
        s[np.arange(past + n)[None] > pos[:, None]] = -np.inf
        w = np.exp(s - s.max(1, keepdims=True))
        ref = (w / w.sum(1, keepdims=True)) @ V[:, h // 2] / (1 + np.exp(-qg[:, h, 1]))
        assert np.abs(og[:, h] - ref).max() < 1e-12


def test_rotation_keeps_angles():
    """Rotated pairs keep their length, and the product of a query and a key depends on their distance only."""
    r = np.random.default_rng(3)
    q, k, w = r.standard_normal((1, 1, 256)), r.standard_normal((1, 1, 256)), np.ones(256)
    rot = lambda x, p: serve.norm_rope(x, w, np.array([p]), 64, 1e6, 0.0)[0, 0]  # noqa: E731
    assert np.allclose(rot(q, 5) @ rot(k, 2), rot(q, 1005) @ rot(k, 1002), atol=1e-9)
    a = rot(q, 77)
    b = rot(q, 0)
    assert np.allclose(a[:32] ** 2 + a[32:64] ** 2, b[:32] ** 2 + b[32:64] ** 2) and np.array_equal(a[64:], b[64:])


def test_plan_form():
    """Every new token has a row of its own in a page of its own request, taken from the end of the stack."""
    past, nnew = [60, 0, 128, 5], [10, 130, 0, 1]
    free = np.arange(20)
    table = np.full((4, 4), -1)
    table[0, 0], table[2, :2], table[3, 0] = 30, [31, 32], 33
    left, t, cu, slot, seq = serve.plan(past, nnew, 145, 4, free, 20, table)
    assert left == 16 and cu.tolist() == [0, 10, 140, 140, 141]
    assert t[0].tolist() == [30, 19, -1, -1] and t[1].tolist() == [18, 17, 16, -1]
    assert slot[:4].tolist() == [30 * 64 + i for i in (60, 61, 62, 63)] and slot[4] == 19 * 64
    assert (slot[141:] == -1).all() and (seq[141:] == -1).all() and len(set(slot[:141])) == 141
