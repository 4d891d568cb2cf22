"""Plain 64-bit forms of the packed-batch operators (include/faie2fn.h section 3c), in numpy: page tables, the 4-bit
cache and its attention, the delta rule over whole prompts."""

import numpy as np

PAGE, HD = 64, 256
LEVELS = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6])
CODES, SCALES = PAGE * HD // 2, PAGE * HD // 32
HEAD_BYTES = 2 * (CODES + SCALES)


def pages(n):
    return (int(n) + PAGE - 1) // PAGE


def plan(past, nnew, T, max_blocks, free, top, table):
    """(free count left, table, cu, slot, seq) of a step, token by token; free is a list used as a stack."""
    table, slot, seq, cu = table.copy(), np.full(T, -1), np.full(T, -1), [0]
    t = 0
    for b, (p, n) in enumerate(zip(past, nnew)):
        n = min(max(int(n), 0), T - t)
        if p >= 0:
            for blk in range(pages(p), min(pages(p + n), max_blocks)):
                table[b, blk] = free[top - 1] if top > 0 else -1
                top = max(top - 1, 0)
        for i in range(n):
            blk = (p + i) // PAGE
            if p >= 0 and blk < max_blocks and table[b, blk] >= 0:
                slot[t] = table[b, blk] * PAGE + (p + i) % PAGE
            seq[t] = b
            t += 1
        cu.append(t)
    return top, table, np.array(cu), slot, seq


def quantise(x):
    """Rows [..., HD] -> (codes [..., HD] of 4 bits, scale bytes [..., HD / 32])."""
    g = np.asarray(x, np.float64).reshape(*np.shape(x)[:-1], HD // 32, 32)
    finite = np.isfinite(g).all(-1)
    g = np.where(finite[..., None], g, 0.0)
    a = np.abs(g).max(-1)
    m, e = np.frexp(a)
    e = np.where(a > 0, np.clip(e - 3 + (m > 0.875), -100, 125), -100)
    u = np.ldexp(np.abs(g), -e[..., None])
    d = np.abs(u[..., None] - LEVELS)
    lo = d.argmin(-1)
    hi = 7 - d[..., ::-1].argmin(-1)        # differs from lo at a tie: the even code of the two
    code = np.where(lo % 2 == 0, lo, hi)
    code = np.where(g < 0, code + 8, code)
    return code.reshape(np.shape(x)).astype(np.uint8), (e + 127).astype(np.uint8)


def values(code, scale):
    v = LEVELS[code & 7] * np.where(code & 8, -1.0, 1.0)
    return v * np.repeat(np.ldexp(1.0, scale.astype(int) - 127), 32, axis=-1)


def offsets():
    """Offset of the byte that holds K's and V's code of (token of a page, dim), and of its scale's byte, by the layout's
    words; and the shift of the code in its byte."""
    t, d = np.meshgrid(np.arange(PAGE), np.arange(HD), indexing="ij")
    g, r = d // 32, d % 32
    kc = np.ravel_multi_index((t // 16, g // 4, g % 4, t % 16, r // 2), (4, 2, 4, 16, 16))
    ks = CODES + np.ravel_multi_index((t // 32, g % 4, t % 16, t % 32 // 16, g // 4), (2, 4, 16, 2, 2))
    key = t % 32 // 16 * 4 + t % 4
    vc = CODES + SCALES + np.ravel_multi_index((t // 32, g // 2, t % 16 // 4, r // 2, g % 2, key), (2, 4, 4, 16, 2, 8))
    vs = 2 * CODES + SCALES + np.ravel_multi_index((t // 32, t % 16 // 4, g, key), (2, 4, 8, 8))
    return kc, ks, vc, vs, 4 * (d % 2)


_OFF = offsets()


def store(cache, slot, k, v):
    """Rows k, v [nkv][HD] into slot of cache [npages][nkv][HEAD_BYTES] (uint8, in place)."""
    kc, ks, vc, vs, sh = (o[slot % PAGE] for o in _OFF)
    for x, c, s in ((k, kc, ks), (v, vc, vs)):
        code, scale = quantise(x)
        for g in range(cache.shape[1]):
            page = cache[slot // PAGE, g]
            page[c[0::2]] = code[g, 0::2] | code[g, 1::2] << 4
            page[s[::32]] = scale[g]


def load(cache, slots):
    """The values of slots: K, V [n][nkv][HD] float64."""
    slots = np.asarray(slots)
    kc, ks, vc, vs, sh = (o[slots % PAGE] for o in _OFF)
    out = []
    for c, s in ((kc, ks), (vc, vs)):
        pg = cache[slots // PAGE]                                     # [n][nkv][HEAD_BYTES]
        code = np.take_along_axis(pg, np.broadcast_to(c[:, None], (len(slots), cache.shape[1], HD)), 2)
        code = code >> sh[:, None].astype(np.uint8) & 15
        scale = np.take_along_axis(pg, np.broadcast_to(s[:, None], code.shape), 2)
        out.append(LEVELS[code & 7] * np.where(code & 8, -1.0, 1.0) * np.ldexp(1.0, scale.astype(int) - 127))
    return out


def norm_rope(x, w, pos, nrot, theta, eps):
    """Rows [n][heads][HD] at positions pos [n]."""
    x = np.asarray(x, np.float64)
    y = x / np.sqrt((x * x).mean(-1, keepdims=True) + np.float64(np.float32(eps))) * np.asarray(w, np.float64)
    h = nrot // 2
    if h:
        ang = np.asarray(pos, np.float64)[:, None] * float(theta) ** (-2.0 * np.arange(h) / nrot)
        c, s = np.cos(ang)[:, None], np.sin(ang)[:, None]
        a, b = y[..., :h].copy(), y[..., h:nrot].copy()
        y[..., :h], y[..., h:nrot] = a * c - b * s, b * c + a * s
    return y


def attn_kv4(past, cu, table, slot, qg, k, v, wq, wk, cache, nrot=64, theta=1e7, eps=1e-6):
    """og [cu[-1]][nq][HD] float64; cache is updated in place."""
    nq, nkv = qg.shape[1], k.shape[1]
    grp, npages = nq // nkv, cache.shape[0]
    og = np.zeros((cu[-1], nq, HD))
    with np.errstate(invalid="ignore", over="ignore"):
        for b, p in enumerate(past):
            rows = np.arange(cu[b], cu[b + 1])
            kn = norm_rope(k[rows], wk, p + rows - cu[b], nrot, theta, eps)
            for i, t in enumerate(rows):
                if slot[t] >= 0:
                    store(cache, int(slot[t]), kn[i], v[t])
        for b, p in enumerate(past):
            rows = np.arange(cu[b], cu[b + 1])
            if p < 0 or not len(rows):
                continue
            pos = p + rows - cu[b]
            q = norm_rope(qg[rows, :, 0], wq, pos, nrot, theta, eps)
            keys = np.arange(min(p + len(rows), table.shape[1] * PAGE))
            page = table[b, keys // PAGE]
            keys, page = keys[(page >= 0) & (page < npages)], page[(page >= 0) & (page < npages)]
            if not len(keys):
                continue
            K, V = load(cache, page * PAGE + keys % PAGE)
            for i, t in enumerate(rows):
                see = keys <= pos[i]
                if not see.any():
                    continue
                for h in range(nq):
                    s = K[see, h // grp] @ q[i, h] / np.sqrt(HD)
                    w = np.exp(s - s.max())
                    og[t, h] = w @ V[see, h // grp] / w.sum()
            og[rows] /= 1.0 + np.exp(-np.asarray(qg[rows, :, 1], np.float64))
    return og
