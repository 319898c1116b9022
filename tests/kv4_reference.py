"""The 4-bit paged cache, its attention and the sampler in numpy, 64 bits, from their definitions."""
import numpy as np

GROUP, STEP_MAX, HALF_MAX, ONE = 64, 4366.0, 65504.0, 2.0 ** 40


def pack_rows(code):
    """Codes [..., d] -> bytes [..., d/2]: 32-bit words, word j of group j % g, elements 8 * (j // g) .. + 7."""
    d = code.shape[-1]
    g = d // GROUP
    out = np.zeros(code.shape[:-1] + (d // 2,), np.uint8)
    for e in range(d):
        grp, i = divmod(e, GROUP)
        word = (i // 8) * g + grp
        out[..., 4 * word + (i % 8) // 2] |= (code[..., e].astype(np.uint8) << (4 * (i % 2))).astype(np.uint8)
    return out


def unpack_rows(b):
    d = 2 * b.shape[-1]
    g = d // GROUP
    out = np.zeros(b.shape[:-1] + (d,), np.uint8)
    for e in range(d):
        grp, i = divmod(e, GROUP)
        word = (i // 8) * g + grp
        out[..., e] = (b[..., 4 * word + (i % 8) // 2] >> (4 * (i % 2))) & 15
    return out


def values(codes, params):
    """Rows of the cache as float64 [..., d]."""
    c = unpack_rows(codes).astype(np.float64)
    p = params.astype(np.float64)
    return c * np.repeat(p[..., 0], GROUP, -1) + np.repeat(p[..., 1], GROUP, -1)


def quantise(x):
    """(codes [..., d], params [..., d/64, 2] fp16) of x [..., d], in x's own precision."""
    g = x.reshape(x.shape[:-1] + (-1, GROUP))
    lo, hi = g.min(-1), g.max(-1)
    m = np.clip(lo, -HALF_MAX, HALF_MAX).astype(np.float16)
    s = np.minimum((hi - lo) * x.dtype.type(np.float32(1) / np.float32(15)), x.dtype.type(STEP_MAX)).astype(np.float16)
    sf, mf = s.astype(x.dtype)[..., None], m.astype(x.dtype)[..., None]
    with np.errstate(divide="ignore", invalid="ignore"):
        c = np.where(sf > 0, np.clip(np.rint((g - mf) / sf), 0, 15), 0)
    return c.astype(np.uint8).reshape(x.shape), np.stack([s, m], -1)


def rope_table(theta, d, n):
    ang = np.arange(n, dtype=np.float64)[:, None] * theta ** (-2.0 * np.arange(d // 2) / d)
    return np.stack([np.cos(ang), np.sin(ang)], -1).astype(np.float32)


def norm_rotate(x, w, cs, eps):
    """x [rows, heads, d] normalised per head (w or None) and rotated, in x's precision."""
    if w is not None:
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + x.dtype.type(eps)) * w.astype(x.dtype)
    c, s = cs[:, None, :, 0].astype(x.dtype), cs[:, None, :, 1].astype(x.dtype)
    h = x.shape[-1] // 2
    a, b = x[..., :h], x[..., h:]
    return np.concatenate([a * c - b * s, b * c + a * s], -1)


def attention(q, cache, table, row_start, ctx_len, nq, nkv, d, scale=None, bad_pages=()):
    """q [rows, nq * d] float64; cache = numpy (k_codes, k_params, v_codes, v_params)."""
    kc, kp, vc, vp = cache
    page = kc.shape[2]
    scale = 1 / np.sqrt(d) if scale is None else scale
    out = np.zeros_like(q)
    for b, ctx in enumerate(ctx_len):
        n = row_start[b + 1] - row_start[b]
        pos = np.arange(max(0, ctx))
        pos = pos[pos // page < table.shape[1]]
        pg = table[b][pos // page] if len(pos) else np.zeros(0, int)
        pos = pos[(pg >= 0) & (pg < kc.shape[0])]
        pg = table[b][pos // page] if len(pos) else pg[:0]
        k = values(kc[pg, :, pos % page], kp[pg, :, pos % page]) if len(pos) else np.zeros((0, nkv, d))
        v = values(vc[pg, :, pos % page], vp[pg, :, pos % page]) if len(pos) else np.zeros((0, nkv, d))
        for r in range(n):
            row = row_start[b] + r
            see = pos <= ctx - n + r
            if not see.any():
                continue
            for h in range(nq):
                s = scale * (k[see, h // (nq // nkv)] @ q[row, h * d:(h + 1) * d])
                p = np.exp(s - s.max())
                out[row, h * d:(h + 1) * d] = p @ v[see, h // (nq // nkv)] / p.sum()
    return out


def sample_kept(x, t, k, top_p, min_p):
    """(weights among the kept tokens in index order, order of tokens) of one row of logits, 64 bits."""
    x = np.where(np.isnan(x), -np.inf, x.astype(np.float64))
    top = x.max()
    if not t > 0:
        t, k = 1.0, 1
    with np.errstate(invalid="ignore"):
        z = np.where(x == top, 0.0, (x - top) / t)
    w = np.floor(np.exp(z) * ONE)
    order = np.argsort(-z, kind="stable")
    ws = w[order]
    if min_p > 0:
        ws[ws < min_p * ONE] = 0
    if k > 0:
        ws[k:] = 0
    if top_p < 1:
        before = np.cumsum(ws) - ws
        cut = before >= np.ceil(top_p * ws.sum())
        cut[0] = False
        ws[cut] = 0
    kept = np.zeros_like(w)
    kept[order] = ws
    return kept, order
