"""Performance cases of the operators that serve a batch of requests of different lengths: the page tables of a paged
cache, attention over that cache held in 4 bits, and the gated delta rule over whole prompts.

The tokens of a batch are packed: request b has rows cu[b] .. cu[b + 1] - 1 of every per-token tensor.  `own` false
computes the operators in plain torch; true makes the library's calls.
"""

import math
import os
import random
import sys

import numpy as np
import torch

own = False

DEV = "cuda"
HD = 256           # head dimension of the attention layers
DK = 128           # head dimension of the DeltaNet layers
NROT, THETA = 64, 1e7
EPS = float(np.float32(1e-6))
PAGE = 64          # tokens a page
CHUNK = 64
LEVELS = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)  # magnitudes of a 4-bit value (e2m1); bit 3 is the sign
HEAD_BYTES = 2 * (PAGE * HD // 2 + PAGE * HD // 32)  # a page of one key/value head: codes and scales of K, then of V

_fn = None


def lib():
    global _fn
    if _fn is None:
        sys.path.insert(0, os.path.join(os.getcwd(), "faie2-flashnext_amd"))
        torch.cuda.init()  # torch first: the library then uses the HIP runtime that torch has loaded
        import fn
        _fn = fn.FN()
    return _fn


def listed():
    return [
        # the tables of a decode step of a small server: one new token a request
        dict(name="plan_decode_b16", kind="plan", B=16, past=8000, new=1, shape="ragged", lens=1),
        # the tables of a step of a large server that decodes most requests and takes in prompts beside them
        dict(name="plan_mixed_b512", kind="plan", B=512, past=16000, new=500, shape="mixed", lens=2),
        # decode of one user, a short context: the latency of the smallest call
        dict(name="attn_b1_4k", kind="attn", B=1, past=4095, new=1, nq=16, nkv=2, shape="even", lens=0),
        # decode of a batch of long contexts of different lengths
        dict(name="attn_b16_32k", kind="attn", B=16, past=32767, new=1, nq=16, nkv=2, shape="ragged", lens=3),
        # decode of a full batch
        dict(name="attn_b64_8k", kind="attn", B=64, past=8191, new=1, nq=16, nkv=2, shape="even", lens=0),
        # a verify step: four drafted tokens a request, the reference model's heads
        dict(name="attn_verify_b8_16k", kind="attn", B=8, past=16380, new=4, nq=24, nkv=2, shape="ragged", lens=4),
        # a whole prompt of one request
        dict(name="attn_prompt_4k", kind="attn", B=1, past=0, new=4001, nq=16, nkv=2, shape="even", lens=0),
        # a serving step that decodes most of its requests and takes in pieces of prompts beside them
        dict(name="attn_mixed_b24", kind="attn", B=24, past=8000, new=300, nq=16, nkv=4, shape="mixed", lens=5),
        # the delta rule over one long prompt
        dict(name="core_b1_15k", kind="core", B=1, past=0, new=15000, nkh=16, nvh=32, head_map=0, shape="even", lens=0),
        # the delta rule over a batch of short prompts
        dict(name="core_b32_short", kind="core", B=32, past=0, new=330, nkh=16, nvh=32, head_map=1, shape="ragged", lens=6),
        # a whole DeltaNet layer step over one prompt, the reference model's heads
        dict(name="block_b1_4k", kind="block", B=1, past=0, new=4096, nkh=16, nvh=48, head_map=0, gate_act=0,
             shape="even", lens=0),
        # the same over a few prompts, some of them continued
        dict(name="block_b4_1k", kind="block", B=4, past=700, new=1100, nkh=16, nvh=32, head_map=1, gate_act=1,
             shape="ragged", lens=7),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["plan", "attn", "attn", "attn", "core", "core", "block"])
    shape = rng.choice(["even", "ragged", "ragged", "mixed"])
    lens = rng.randint(1, 1 << 20)
    if kind == "plan":
        return dict(kind=kind, B=_log(rng, 1, 1000), past=_log(rng, 1, 30000), new=_log(rng, 1, 500), shape=shape, lens=lens)
    if kind == "attn":
        nq, nkv = rng.choice([(16, 2), (16, 2), (24, 2), (16, 4), (8, 2), (8, 8)])
        if rng.random() < 0.6:  # decode and verify steps
            B = _log(rng, 1, 64)
            past, new = _log(rng, 1, min(100000, 1000000 // (B * nkv))), rng.choice([1, 1, 1, 2, 3, 4, 8])
        else:  # prompts, whole or in pieces
            B, new = _log(rng, 1, 8), _log(rng, 9, 1500)
            new = max(9, new // B)
            past = rng.choice([0, _log(rng, 1, 2000)])
        return dict(kind=kind, B=B, past=past, new=new, nq=nq, nkv=nkv, shape=shape, lens=lens)
    B = _log(rng, 1, 40)
    nvh = rng.choice([16, 32, 48])
    new = _log(rng, 1, (10000 if kind == "core" else 4000) // B)
    c = dict(kind=kind, B=B, past=rng.choice([0, rng.randint(1, 5000)]), new=new, nkh=16, nvh=nvh,
             head_map=rng.randint(0, 1), shape=shape, lens=lens)
    return dict(c, gate_act=rng.randint(0, 1)) if kind == "block" else c


# ---- inputs ----

def _lengths(c):
    """Tokens behind and new tokens of each request."""
    r = random.Random(c["lens"])
    past, new = [c["past"]] * c["B"], [c["new"]] * c["B"]
    for b in range(1, c["B"]):
        if c["shape"] != "even":
            past[b] = int(c["past"] * r.uniform(0.1, 1.0))
        if c["shape"] == "ragged" and c["new"] > 8:
            new[b] = max(1, int(c["new"] * r.uniform(0.1, 1.0)))
        if c["shape"] == "mixed" and r.random() < 0.75:
            new[b] = 1
    return past, new


def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(int(seed))
    return g


def _n(g, *shape, mean=0.0, std=1.0):
    t = torch.randn(shape, generator=g, device=DEV)
    return t if mean == 0.0 and std == 1.0 else t.mul_(std).add_(mean)


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def _pages(n):
    return (n + PAGE - 1) // PAGE


def _batch(c, g):
    """The request tables of a step, as the page plan leaves them: pages in random order."""
    past, new = _lengths(c)
    B = c["B"]
    cu = [0]
    for n in new:
        cu.append(cu[-1] + n)
    want = [_pages(p + n) for p, n in zip(past, new)]
    npages, mb = sum(want) + 7, max(want) + 1
    order = torch.randperm(npages, generator=g, device=DEV).int()
    s = dict(B=B, T=cu[-1], npages=npages, mb=mb, past=_i32(past), cu=_i32(cu))
    lp, ln = s["past"].long(), _i32(new).long()
    ends = torch.cumsum(_pages(lp + ln), 0)
    j = torch.arange(mb, device=DEV)
    at = (ends - _pages(lp + ln))[:, None] + j
    s["table"] = torch.where(j < _pages(lp + ln)[:, None], order[at.clamp(max=npages - 1)], -1).int().contiguous()
    s["seq"] = torch.repeat_interleave(torch.arange(B, device=DEV), ln).int()
    own_seq = s["seq"].long()
    p = lp[own_seq] + torch.arange(s["T"], device=DEV) - s["cu"].long()[own_seq]
    s["slot"] = (s["table"][own_seq, p // PAGE] * PAGE + p % PAGE).int()
    return s


def _plan_inputs(c, seed):
    g = _gen(seed)
    past, new = _lengths(c)
    have, want = [_pages(p) for p in past], [_pages(p + n) for p, n in zip(past, new)]
    npages, mb, T = sum(want) + 64, max(want) + 1, sum(new)
    order = torch.randperm(npages, generator=g, device=DEV).int()
    j = torch.arange(mb, device=DEV)
    h = _i32(have).long()
    at = (torch.cumsum(h, 0) - h)[:, None] + j
    table = torch.where(j < h[:, None], order[at.clamp(max=npages - 1)], -1).int().contiguous()
    top = npages - sum(have)
    free = torch.full((npages,), -1, dtype=torch.int32, device=DEV)
    free[:top] = order[sum(have):]
    return dict(T=T, npages=npages, mb=mb, past=_i32(past), new=_i32(new), free=free, top=_i32([top]), table=table,
                left=_i32([0]), cu=torch.empty(c["B"] + 1, dtype=torch.int32, device=DEV),
                slot=torch.empty(T, dtype=torch.int32, device=DEV), seq=torch.empty(T, dtype=torch.int32, device=DEV))


def _codes(g, n):
    """n bytes of two 4-bit values each, distributed as the codes of normal values are."""
    pairs = torch.linspace(0.5 / 256, 1 - 0.5 / 256, 256, dtype=torch.float64)
    a = torch.erfinv(2 * pairs - 1) * math.sqrt(2) / 0.5  # normal values over a scale of 1/2
    mid = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], dtype=torch.float64)
    code = torch.bucketize(a.abs(), mid) + 8 * (a < 0).long()
    table = (code[:, None] + 16 * code[None, :]).reshape(-1).to(torch.uint8).to(DEV)
    out = torch.empty(n, dtype=torch.uint8, device=DEV)
    for i in range(0, n, 1 << 26):
        m = min(1 << 26, n - i)
        out[i:i + m] = table[torch.randint(0, 65536, (m,), generator=g, device=DEV, dtype=torch.int32)]
    return out


def _attn_inputs(c, seed):
    g = _gen(seed)
    s = _batch(c, g)
    T, nq, nkv = s["T"], c["nq"], c["nkv"]
    half = HEAD_BYTES // 2
    cache = torch.empty(s["npages"], nkv, 2, half, dtype=torch.uint8, device=DEV)
    cut = PAGE * HD // 2
    cache[..., :cut] = _codes(g, s["npages"] * nkv * 2 * cut).reshape(s["npages"], nkv, 2, cut)
    cache[..., cut:] = torch.randint(125, 127, (s["npages"], nkv, 2, half - cut), generator=g, device=DEV, dtype=torch.uint8)
    s.update(cache=cache.reshape(s["npages"], nkv, HEAD_BYTES), qg=_n(g, T, nq, 2, HD), k=_n(g, T, nkv, HD),
             v=_n(g, T, nkv, HD), wq=_n(g, HD, mean=1.0, std=0.1), wk=_n(g, HD, mean=1.0, std=0.1),
             og=torch.empty(T, nq, HD, device=DEV), kn=torch.empty(T, nkv, HD, device=DEV),
             vn=torch.empty(T, nkv, HD, device=DEV))
    return s


def _gdn_inputs(c, seed):
    g = _gen(seed)
    past, new = _lengths(c)
    B, T, nkh, nvh = c["B"], sum(new), c["nkh"], c["nvh"]
    cu = [0]
    for n in new:
        cu.append(cu[-1] + n)
    s = dict(B=B, T=T, cu=_i32(cu), S=_n(g, B, nvh, DK, DK, std=0.05), out=torch.empty(T, nvh, DK, device=DEV))
    if c["kind"] == "core":
        unit = lambda x: x.div_(x.norm(dim=-1, keepdim=True))  # noqa: E731
        s.update(q=unit(_n(g, T, nkh, DK)), k=unit(_n(g, T, nkh, DK)), v=_n(g, T, nvh, DK),
                 beta=torch.sigmoid(_n(g, T, nvh)),
                 g=-torch.exp(_n(g, nvh, std=0.5)) * torch.nn.functional.softplus(_n(g, T, nvh)))
    else:
        C = 2 * nkh * DK + nvh * DK
        s.update(pos=_i32(past), qkv=_n(g, T, C), conv_w=_n(g, C, 4, std=0.3), conv=_n(g, B, 4, C), ab=_n(g, T, 2 * nvh),
                 dt_bias=_n(g, nvh, std=0.5), ssm_a=-torch.exp(_n(g, nvh, std=0.5)), z=_n(g, T, nvh * DK),
                 norm_w=_n(g, DK, mean=1.0, std=0.1))
    return s


def prepare(case, seed):
    c = case
    s = _plan_inputs(c, seed) if c["kind"] == "plan" else \
        _attn_inputs(c, seed) if c["kind"] == "attn" else _gdn_inputs(c, seed)
    s["case"] = c
    past, new = _lengths(c)
    if own and c["kind"] == "attn":
        L = lib()
        s["nsplit"] = L.attn_kv4_nsplit(s["B"], s["T"], c["nq"], c["nkv"], max(p + n for p, n in zip(past, new)))
        s["wb"] = L.attn_kv4_work_bytes(s["B"], s["T"], c["nq"], c["nkv"], s["nsplit"])
    elif own and c["kind"] != "plan":
        s["wb"] = lib().gdn_chunk_work_bytes(s["B"], s["T"], c["nkh"], c["nvh"], c["kind"] == "block")
    if "wb" in s:
        s["work"] = torch.empty(max(16, s["wb"]), dtype=torch.uint8, device=DEV)
    s["lengths"] = (past, new)
    torch.cuda.synchronize()
    return s


# ---- the library's calls ----

def _p(*tensors):
    return [t.data_ptr() for t in tensors]


def _run_own(s):
    c, L, st = s["case"], lib(), torch.cuda.current_stream().cuda_stream
    if c["kind"] == "plan":
        L.page_plan_dev(c["B"], s["T"], s["mb"], s["npages"], *_p(s["past"], s["new"], s["free"], s["top"], s["left"],
                        s["table"], s["cu"], s["slot"], s["seq"]), stream=st)
        return [s["left"], s["table"], s["cu"], s["slot"], s["seq"]]
    if c["kind"] == "attn":
        L.attn_kv4_dev(s["B"], s["T"], c["nq"], c["nkv"], s["mb"], s["npages"], *_p(s["past"], s["cu"], s["table"],
                       s["slot"], s["seq"], s["qg"], s["k"], s["v"], s["wq"], s["wk"], s["cache"]), s["nsplit"],
                       s["work"].data_ptr(), s["wb"], s["og"].data_ptr(), stream=st)
        L.kv4_unpack_dev(s["T"], c["nkv"], s["npages"], *_p(s["slot"], s["cache"], s["kn"], s["vn"]), stream=st)
        return [s["og"], s["kn"], s["vn"]]
    if c["kind"] == "core":
        L.gdn_core_chunk_dev(s["B"], s["T"], c["nkh"], c["nvh"], *_p(s["cu"], s["q"], s["k"], s["v"], s["beta"], s["g"],
                             s["S"], s["out"], s["work"]), s["wb"], stream=st, head_map=c["head_map"])
        return [s["out"], s["S"]]
    L.gdn_block_chunk_dev(s["B"], s["T"], c["nkh"], c["nvh"], 4, *_p(s["cu"], s["pos"], s["qkv"], s["conv_w"], s["conv"],
                          s["ab"], s["dt_bias"], s["ssm_a"], s["S"], s["z"], s["norm_w"], s["out"], s["work"]), s["wb"],
                          stream=st, head_map=c["head_map"], gate_act=c["gate_act"])
    return [s["out"], s["S"], s["conv"]]


# ---- the plain forms ----

def _plan_plain(s):
    B, T = s["past"].numel(), s["T"]
    past, new = s["past"].long(), s["new"].long()
    cu = torch.zeros(B + 1, dtype=torch.long, device=DEV)
    cu[1:] = torch.cumsum(new, 0)
    have, want = _pages(past), _pages(past + new)
    fresh = want - have
    before = torch.cumsum(fresh, 0) - fresh
    j = torch.arange(s["mb"], device=DEV)
    at = s["top"].long() - 1 - (before[:, None] + j - have[:, None])
    fill = (j >= have[:, None]) & (j < want[:, None])
    table = torch.where(fill, s["free"][at.clamp(0, s["npages"] - 1)], s["table"])
    t = torch.arange(T, device=DEV)
    seq = torch.searchsorted(cu, t, right=True) - 1
    p = past[seq] + t - cu[seq]
    s["table"].copy_(table)
    return [(s["top"] - fresh.sum()).int(), s["table"], cu.int(), (table[seq, p // PAGE] * PAGE + p % PAGE).int(), seq.int()]


def _quantise(y):
    """Values [..., HD] in float64 -> (codes, scale exponents): groups of 32 share the least power of two that leaves
    their largest value off by at most half a step."""
    y = y.reshape(*y.shape[:-1], HD // 32, 32)
    m, e = torch.frexp(y.abs().amax(-1))
    e = torch.where(m == 0, -100, (e - 3 + (m > 0.875).int()).clamp(-100, 125)).int()
    a = torch.ldexp(y.abs(), -e[..., None])
    code = torch.zeros(y.shape, dtype=torch.uint8, device=DEV)
    for level, up in ((0.25, False), (0.75, True), (1.25, False), (1.75, True), (2.5, False), (3.5, True), (5.0, False)):
        code += (a >= level) if up else (a > level)
    return code + 8 * (y < 0).to(torch.uint8), e


def _values(code, e):
    level = torch.tensor(LEVELS, device=DEV)
    v = level[(code & 7).long()] * (1 - 2 * (code >> 3).float())
    return torch.ldexp(v, e[..., None]).reshape(*code.shape[:-2], HD)


def _rows_of_pages(pages):
    """Pages [n][nkv][HEAD_BYTES] -> K, V [n * PAGE][nkv][HD] float32."""
    n, nkv, _ = pages.shape
    cut, half = PAGE * HD // 2, HEAD_BYTES // 2
    level = torch.tensor([x * sign for sign in (1, -1) for x in LEVELS], device=DEV)

    def nibbles(b):
        return torch.stack([level[(b & 15).long()], level[(b >> 4).long()]], -1)

    # K: 16-key blocks, halves of the row, groups of the half, keys, the group's dims
    k = nibbles(pages[..., :cut].reshape(n, nkv, 4, 2, 4, 16, 16)).reshape(n, nkv, 4, 2, 4, 16, 32)
    k = k.permute(0, 2, 5, 1, 3, 4, 6).reshape(n * PAGE, nkv, 8, 32)
    # its scales: 32-key blocks, groups of the half, keys, 16-key block, half of the row
    ks = pages[..., cut:half].reshape(n, nkv, 2, 4, 16, 2, 2).permute(0, 2, 5, 4, 1, 6, 3).reshape(n * PAGE, nkv, 8)
    # V: 32-key blocks, pairs of groups, quarters, pairs of dims, group of the pair, 16-key block, key of the quarter
    v = nibbles(pages[..., half:half + cut].reshape(n, nkv, 2, 4, 4, 16, 2, 2, 4))
    v = v.permute(0, 2, 7, 4, 8, 1, 3, 6, 5, 9).reshape(n * PAGE, nkv, 8, 32)
    vs = pages[..., half + cut:].reshape(n, nkv, 2, 4, 8, 2, 4).permute(0, 2, 5, 3, 6, 1, 4).reshape(n * PAGE, nkv, 8)
    return [torch.ldexp(x, e[..., None].int() - 127).reshape(n * PAGE, nkv, HD) for x, e in ((k, ks), (v, vs))]


def _norm_rope(x, w, pos):
    """RMSNorm and the rotation of the first NROT dims by pos * THETA^(-2i/NROT), in float64."""
    x = x.double()
    y = x / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS) * w.double()
    i = torch.arange(NROT // 2, device=DEV, dtype=torch.float64)
    ang = (pos.double()[:, None] * THETA ** (-2.0 * i / NROT))[:, None]
    cs, sn, h = torch.cos(ang), torch.sin(ang), NROT // 2
    return torch.cat([y[..., :h] * cs - y[..., h:NROT] * sn, y[..., h:NROT] * cs + y[..., :h] * sn, y[..., NROT:]], -1)


def _attn_plain(s):
    c = s["case"]
    nq, nkv = c["nq"], c["nkv"]
    grp = nq // nkv
    seq = s["seq"].long()
    pos = s["past"].long()[seq] + torch.arange(s["T"], device=DEV) - s["cu"].long()[seq]
    kn = _values(*_quantise(_norm_rope(s["k"], s["wk"], pos)))
    vn = _values(*_quantise(s["v"].double()))
    q = _norm_rope(s["qg"][:, :, 0], s["wq"], pos).float()
    gate = torch.sigmoid(s["qg"][:, :, 1])
    og = torch.empty(s["T"], nq, HD, device=DEV)
    t0 = 0
    for b, (p, n) in enumerate(zip(*s["lengths"])):
        K, V = _rows_of_pages(s["cache"][s["table"][b, :_pages(p + n)].long()])
        K[p:p + n], V[p:p + n] = kn[t0:t0 + n], vn[t0:t0 + n]
        K, V = K[:p + n].permute(1, 2, 0).contiguous(), V[:p + n].permute(1, 0, 2).contiguous()
        for i in range(0, n, 512):
            m = min(512, n - i)
            e = p + i + m
            sc = q[t0 + i:t0 + i + m].reshape(m, nkv, grp, HD).permute(1, 0, 2, 3).reshape(nkv, m * grp, HD) @ K[..., :e]
            sc = (sc / math.sqrt(HD)).reshape(nkv, m, grp, e)
            if m > 1:
                far = torch.arange(e, device=DEV) > p + i + torch.arange(m, device=DEV)[:, None]
                sc.masked_fill_(far[None, :, None], -math.inf)
            w = torch.exp(sc - sc.amax(-1, keepdim=True))
            w /= w.sum(-1, keepdim=True)
            o = (w.reshape(nkv, m * grp, e) @ V[:, :e]).reshape(nkv, m, grp, HD)
            og[t0 + i:t0 + i + m] = o.permute(1, 0, 2, 3).reshape(m, nq, HD)
        t0 += n
    return [og * gate, kn, vn]


def _heads(c):
    h = torch.arange(c["nvh"], device=DEV)
    return h // (c["nvh"] // c["nkh"]) if c["head_map"] else h % c["nkh"]


def _delta_plain(c, s, q, k, v, beta, g):
    """The delta rule chunk by chunk: in a chunk the updates u solve a triangular system, so that only the state
    between chunks is sequential."""
    heads, nvh = _heads(c), c["nvh"]
    out = torch.empty_like(v)
    eye = torch.eye(CHUNK, device=DEV)
    t0 = 0
    for b, n in enumerate(s["lengths"][1]):
        N = (n + CHUNK - 1) // CHUNK

        def chunks(x):  # [n][heads][...] -> [heads][N][CHUNK][...]
            pad = torch.zeros(N * CHUNK - n, *x.shape[1:], device=DEV, dtype=x.dtype)
            x = torch.cat([x[t0:t0 + n], pad]).transpose(0, 1)
            return x.reshape(x.shape[0], N, CHUNK, *x.shape[2:]).contiguous()

        Q, K, V, be = chunks(q)[heads], chunks(k)[heads], chunks(v), chunks(beta)
        G = torch.cumsum(chunks(g).double(), -1)
        D = torch.tril(torch.exp(torch.tril(G[..., :, None] - G[..., None, :]))).float()
        eg, last = torch.exp(G).float()[..., None], torch.exp(G[..., -1:] - G).float()[..., None]
        Kt = K.transpose(-1, -2).contiguous()
        A = torch.tril(be[..., None] * D * (K @ Kt), -1)
        inv = eye.expand(nvh, N, CHUNK, CHUNK).clone()
        for i in range(1, CHUNK):
            inv[..., i, :] -= (A[..., i, :i, None] * inv[..., :i, :]).sum(-2)
        W, U0 = inv @ (be[..., None] * eg * K), inv @ (be[..., None] * V)
        P = D * (Q @ Kt)
        Q, Kt, St = Q * eg, Kt * last.transpose(-1, -2), s["S"][b]
        o = torch.empty_like(V)
        for i in range(N):
            U = U0[:, i] - W[:, i] @ St
            o[:, i] = Q[:, i] @ St + P[:, i] @ U
            St = eg[:, i, -1:] * St + Kt[:, i] @ U
        s["S"][b] = St
        out[t0:t0 + n] = o.reshape(nvh, N * CHUNK, DK)[:, :n].transpose(0, 1) / math.sqrt(DK)
        t0 += n
    return out


def _block_plain(c, s):
    T, nkh, nvh, ring = s["T"], c["nkh"], c["nvh"], 4
    x, conv = s["qkv"], s["conv"]
    y = x * s["conv_w"][:, 3]
    t0 = 0
    for b, (p, n) in enumerate(zip(*s["lengths"])):
        hist = torch.cat([conv[b, [(p - d) % ring for d in (3, 2, 1)]], x[t0:t0 + n]])
        for j in range(3):
            y[t0:t0 + n] += hist[j:j + n] * s["conv_w"][:, j]
        for d in range(1, min(3, n) + 1):
            conv[b, (p + n - d) % ring] = x[t0 + n - d]
        t0 += n
    y = y * torch.sigmoid(y)
    q, k = (a.reshape(T, nkh, DK) for a in (y[:, :nkh * DK], y[:, nkh * DK:2 * nkh * DK]))
    q, k = (a / torch.sqrt((a * a).sum(-1, keepdim=True) + EPS) for a in (q, k))
    sp = s["ab"][:, :nvh] + s["dt_bias"]
    sp = torch.where(sp > 20, sp, torch.log1p(torch.exp(sp)))
    o = _delta_plain(c, s, q.contiguous(), k.contiguous(), y[:, 2 * nkh * DK:].reshape(T, nvh, DK),
                     torch.sigmoid(s["ab"][:, nvh:]), sp * s["ssm_a"])
    z = s["z"].reshape(T, nvh, DK)
    gate = torch.sigmoid(z) * z if c["gate_act"] else torch.sigmoid(z)
    return [o / torch.sqrt((o * o).mean(-1, keepdim=True) + EPS) * s["norm_w"] * gate, s["S"], conv]


def run(state):
    s = state
    if own:
        return _run_own(s)
    kind = s["case"]["kind"]
    if kind == "plan":
        return _plan_plain(s)
    if kind == "attn":
        return _attn_plain(s)
    if kind == "core":
        return [_delta_plain(s["case"], s, s["q"], s["k"], s["v"], s["beta"], s["g"]), s["S"]]
    return _block_plain(s["case"], s)


# ---- the work a pass cannot do without ----

def work(case):
    c = case
    past, new = _lengths(c)
    T = sum(new)
    if c["kind"] == "plan":
        fresh = sum(_pages(p + n) - _pages(p) for p, n in zip(past, new))
        return dict(bytes=4 * (2 * c["B"] + c["B"] + 1 + 2 * fresh + 2 * T + 2), flops=4 * T)
    if c["kind"] == "attn":
        keys = sum(p + n for p, n in zip(past, new))
        seen = sum(n * p + n * (n + 1) // 2 for p, n in zip(past, new))
        head = 2 * (HD // 2 + HD // 32)  # a cached key and value of one head
        return dict(bytes=c["nkv"] * head * (keys + T) + 4 * HD * T * (3 * c["nq"] + 2 * c["nkv"]) + 4 * HD * T * 2 * c["nkv"],
                    flops=4 * HD * c["nq"] * seen)
    nkh, nvh = c["nkh"], c["nvh"]
    b = 4 * c["B"] * nvh * DK * DK * 2 + 4 * T * (2 * nkh * DK + 2 * nvh * DK + 2 * nvh)
    if c["kind"] == "block":
        C = 2 * nkh * DK + nvh * DK
        b += 4 * T * nvh * DK + 4 * C * (4 + 6 * c["B"])
    return dict(bytes=b, flops=8 * T * nvh * DK * DK)


# ---- the same in 64 bits, from the definitions ----

def _plan_exact(c, s):
    past, new = _lengths(c)
    free, top, table = s["free"].tolist(), int(s["top"]), s["table"].tolist()
    cu, slot, seq = [0], [], []
    for b, (p, n) in enumerate(zip(past, new)):
        for i in range(p, p + n):
            if i % PAGE == 0:
                top -= 1
                table[b][i // PAGE] = free[top]
            slot.append(table[b][i // PAGE] * PAGE + i % PAGE)
            seq.append(b)
        cu.append(len(slot))
    return [_i32([top]), _i32(table), _i32(cu), _i32(slot), _i32(seq)]


def _page_offsets():
    """Byte offset and shift of the code, and byte offset of the scale, of each (token of a page, dim) of K and of V."""
    t, d = np.meshgrid(np.arange(PAGE), np.arange(HD), indexing="ij")
    grp, r = d // 32, d % 32
    kb = (((t // 16 * 2 + grp // 4) * 4 + grp % 4) * 16 + t % 16) * 16 + r // 2
    lane = t % 16 // 4 * 16 + r // 2
    vb = ((t // 32 * 4 + grp // 2) * 64 + lane) * 16 + grp % 2 * 8 + t % 32 // 16 * 4 + t % 4
    cut, half = PAGE * HD // 2, HEAD_BYTES // 2
    ks = cut + ((t // 32 * 4 + grp % 4) * 16 + t % 16) * 4 + t % 32 // 16 * 2 + grp // 4
    vs = half + cut + ((t // 32 * 4 + t % 16 // 4) * 8 + grp) * 8 + t % 32 // 16 * 4 + t % 4
    return [torch.from_numpy(x).to(DEV) for x in (kb, 4 * (d % 2), ks, half + vb, 4 * (d % 2), vs)]


def _nearest(x):
    """Rows [n][nkv][HD] float64 -> the values that their 4-bit form stands for."""
    a = x.abs().reshape(-1, 32)
    big = a.amax(1)
    e = torch.floor(torch.log2(torch.where(big > 0, big, 1.0)))
    e = torch.where(2.0 ** e > big, e - 1, e)
    e = torch.where(2.0 ** (e + 1) <= big, e + 1, e) - 2
    e = torch.where(big > 7 * 2.0 ** e, e + 1, e)
    step = (2.0 ** torch.where(big > 0, e, -100).clamp(-100, 125))[:, None]
    u = a / step
    r = torch.where(u <= 2, torch.round(2 * u) / 2, torch.where(u <= 4, torch.round(u), 2 * torch.round(u / 2))).clamp(max=6)
    return (r * step).reshape(x.shape) * torch.sign(x)


def _attn_exact(c, s):
    past, new = _lengths(c)
    nq, nkv = c["nq"], c["nkv"]
    grp = nq // nkv
    if 4 * HD * nq * sum(n * (p + n) for p, n in zip(past, new)) > 3e13:
        return None
    koff, ksh, kse, voff, vsh, vse = _page_offsets()
    level = torch.tensor([x * sign for sign in (1.0, -1.0) for x in LEVELS], dtype=torch.float64, device=DEV)
    i = torch.arange(NROT // 2, dtype=torch.float64, device=DEV)

    def turned(x, w, at):  # [n][heads][HD] at positions `at`
        x = x.double()
        y = w.double() * x * torch.rsqrt((x ** 2).sum(-1, keepdim=True) / HD + EPS)
        z = torch.exp(1j * at.double()[:, None, None] * THETA ** (-i / (NROT // 2)))
        r = torch.complex(y[..., :NROT // 2].contiguous(), y[..., NROT // 2:NROT].contiguous()) * z
        return torch.cat([r.real, r.imag, y[..., NROT:]], -1)

    ogs, kns, vns = [], [], []
    t0 = 0
    for b, (p, n) in enumerate(zip(past, new)):
        pages = s["cache"][s["table"][b, :_pages(p + n)].long()]

        def cached(off, sh, sc):
            x = level[((pages[:, :, off].int() >> sh.int()) & 15).long()] * 2.0 ** (pages[:, :, sc].double() - 127)
            return x.permute(1, 0, 2, 3).reshape(nkv, -1, HD)[:, :p + n]

        K, V = cached(koff, ksh, kse), cached(voff, vsh, vse)
        at = torch.arange(p, p + n, device=DEV)
        kn = _nearest(turned(s["k"][t0:t0 + n], s["wk"], at))
        vn = _nearest(s["v"][t0:t0 + n].double())
        K[:, p:], V[:, p:] = kn.transpose(0, 1), vn.transpose(0, 1)
        q = turned(s["qg"][t0:t0 + n, :, 0], s["wq"], at)
        o = torch.empty(n, nq, HD, dtype=torch.float64, device=DEV)
        for h in range(nq):
            Kh = K[h // grp].t().contiguous()
            for j in range(0, n, 1024):
                e = min(n, j + 1024)
                sc = q[j:e, h] @ Kh / HD ** 0.5
                sc = torch.where(torch.arange(p + n, device=DEV) <= at[j:e, None], sc, -math.inf)
                o[j:e, h] = torch.softmax(sc, -1) @ V[h // grp]
        ogs.append(o * torch.sigmoid(s["qg"][t0:t0 + n, :, 1].double()))
        kns.append(kn)
        vns.append(vn)
        t0 += n
    return [torch.cat(x) for x in (ogs, kns, vns)]


def _gdn_exact(c, s):
    """Token by token, every request that still has one at once."""
    past, new = _lengths(c)
    B, nkh, nvh, heads = c["B"], c["nkh"], c["nvh"], _heads(c)
    S, cu = s["S"].double(), s["cu"].long()
    out = torch.empty(s["T"], nvh, DK, dtype=torch.float64, device=DEV)
    order = sorted(range(B), key=lambda b: -new[b])
    S = S[order]
    start = cu[:-1][order]
    block = c["kind"] == "block"
    if block:
        conv, w = s["conv"].double()[order], s["conv_w"].double()
        pos = _i32(past).long()[order]
        rows = torch.arange(B, device=DEV)
        hist = [conv[rows, (pos - d) % 4] for d in (3, 2, 1)]
    for t in range(max(new)):
        m = sum(n > t for n in new)  # the first m of `order` have a token t
        at = start[:m] + t
        if block:
            x = s["qkv"][at].double()
            hist = [h[:m] for h in hist] + [x]
            y = sum(h * w[:, j] for j, h in enumerate(hist))
            hist = hist[1:]
            conv[rows[:m], (pos[:m] + t) % 4] = x
            y = y / (1 + torch.exp(-y))
            q, k = y[:, :nkh * DK].reshape(m, nkh, DK), y[:, nkh * DK:2 * nkh * DK].reshape(m, nkh, DK)
            q, k = (a * torch.rsqrt((a ** 2).sum(-1, keepdim=True) + EPS) for a in (q, k))
            v = y[:, 2 * nkh * DK:].reshape(m, nvh, DK)
            a = s["ab"][at].double()
            beta = 1 / (1 + torch.exp(-a[:, nvh:]))
            gamma = torch.exp(s["ssm_a"].double() * torch.nn.functional.softplus(a[:, :nvh] + s["dt_bias"].double()))
        else:
            q, k, v, beta = (s[n][at].double() for n in ("q", "k", "v", "beta"))
            gamma = torch.exp(s["g"][at].double())
        q, k = q[:, heads], k[:, heads]
        M = S[:m] * gamma[..., None, None]
        d = (v - (k[..., None, :] @ M)[..., 0, :]) * beta[..., None]
        M += k[..., None] * d[..., None, :]
        S[:m] = M
        o = (q[..., None, :] @ M)[..., 0, :] / DK ** 0.5
        if block:
            z = s["z"][at].double().reshape(m, nvh, DK)
            o = o * torch.rsqrt((o ** 2).mean(-1, keepdim=True) + EPS) * s["norm_w"].double() / (1 + torch.exp(-z))
            o = o * z if c["gate_act"] else o
        out[at] = o
    back = torch.argsort(torch.tensor(order, device=DEV))
    if not block:
        return [out, S[back]]
    # a ring slot that no token of the call wrote stays; of a longer call only the last three positions are written
    ring = s["conv"].double()
    for j, b in enumerate(order):
        for d in range(1, min(3, new[b]) + 1):
            ring[b, (past[b] + new[b] - d) % 4] = conv[j, (past[b] + new[b] - d) % 4]
    return [out, S[back], ring]


def exact(case, seed):
    if case["kind"] == "plan":
        return _plan_exact(case, _plan_inputs(case, seed))
    if case["kind"] == "attn":
        return _attn_exact(case, _attn_inputs(case, seed))
    return _gdn_exact(case, _gdn_inputs(case, seed))
