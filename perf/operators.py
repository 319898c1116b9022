"""The 4-bit paged KV cache and the sampler, case by case: what a serving loop calls between its matrix products.

Three operators, each reached through ``aethermind_b200.ops``:

* ``append``: q and k of new tokens are normalised for each head (optional), rotated, and k and v are quantised to
  4 bits into their pages; the rows are then read back as the values that the cache stands for.
* ``attend``: causal grouped-query attention of the new rows over the 4-bit cache, for single tokens and for prompts.
* ``sample``: one token per row of logits by temperature, top-k, top-p and min-p, from given uniform numbers.

The cache. K and V each have ``codes`` uint8 [pages, kv heads, page, d/2] and ``params`` fp16 [pages, kv heads, page,
d/64, 2]: a (scale s, minimum m) pair for every 64 elements; an element is m + s * code. A row's bytes are little-endian
32-bit words; word j holds group j % (d/64), elements 8 * (j // (d/64)) + i in nibble i. ``page_table`` [sequences,
pages] names the pages of a sequence, ``row_start`` [sequences + 1] says which rows of the call are its new ones, and
``ctx_len`` how many tokens it has with them: row r of n new ones is at position ctx_len - n + r.

The sampler's weights are whole numbers of 2^-40 of the largest one, so that no sum depends on its order.
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
GROUP = 64            # elements that share a scale and a minimum
EPS = 1e-5
HALF_MAX = 65504.0    # largest fp16
STEP_MAX = 4366.0     # largest scale: 15 steps of it stay inside fp16
ONE = 2.0 ** 40       # the weight of the most likely token


# ------------------------------------------------------------------ cases
def listed():
    return [
        # the next token of one conversation: all latency
        dict(name="append_one", op="append", batch=1, rows=1, ctx=513, nq=32, nkv=8, d=128, page=16, norm=False,
             dtype="bf16"),
        # a decode step of a full batch, for models that normalise q and k
        dict(name="append_batch", op="append", batch=96, rows=1, ctx=4096, nq=64, nkv=8, d=128, page=64, norm=True,
             dtype="bf16"),
        # ragged prompts entering the cache together
        dict(name="append_prompts", op="append", batch=7, rows=2048, ctx=2048, nq=32, nkv=8, d=64, page=16, norm=True,
             dtype="bf16"),
        # a small fp32 model's prompt
        dict(name="append_f32", op="append", batch=3, rows=77, ctx=128, nq=4, nkv=2, d=64, page=32, norm=True,
             dtype="f32"),
        # the next token of one short conversation
        dict(name="attend_one", op="attend", batch=1, rows=1, ctx=513, nq=32, nkv=8, d=128, page=16, dtype="bf16"),
        # the next token of one long conversation: few rows, a long axis
        dict(name="attend_long", op="attend", batch=1, rows=1, ctx=65531, nq=64, nkv=8, d=128, page=64, dtype="bf16"),
        # a decode step of a ragged batch
        dict(name="attend_batch", op="attend", batch=64, rows=1, ctx=8192, nq=32, nkv=8, d=128, page=16, dtype="bf16"),
        # a small fp32 model, a few tokens to verify at once
        dict(name="attend_f32", op="attend", batch=5, rows=3, ctx=509, nq=4, nkv=2, d=64, page=16, dtype="f32"),
        # the last chunk of two long prompts
        dict(name="attend_prompt", op="attend", batch=2, rows=2048, ctx=8192, nq=32, nkv=8, d=128, page=64,
             dtype="bf16"),
        # one conversation's next token
        dict(name="sample_one", op="sample", rows=1, vocab=128256, mix="chat", dtype="bf16"),
        # a batch in which every row has its own settings
        dict(name="sample_batch", op="sample", rows=192, vocab=128256, mix="all", dtype="f32"),
        # a small vocabulary of odd size
        dict(name="sample_small", op="sample", rows=33, vocab=509, mix="all", dtype="f32"),
    ]


HEADS = [(32, 8, 128), (32, 8, 64), (64, 8, 128), (4, 2, 64), (28, 4, 128), (16, 16, 64), (12, 1, 128)]


def draw(rng):
    def size(lo, hi):
        return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))

    op = rng.choice(["append", "attend", "attend", "sample"])
    if op == "sample":
        rows = size(1, 192)
        return dict(op=op, rows=rows, vocab=size(200, 128256), mix=rng.choice(["chat", "all"]),
                    dtype=rng.choice(["bf16", "f32"]))
    nq, nkv, d = rng.choice(HEADS)
    page = rng.choice([16, 32, 64, 128, 256])
    dtype = rng.choice(["bf16", "bf16", "bf16", "f32"])
    if op == "append":
        tokens = 7 * 2048 * 40 * 64 * 2 // ((nq + nkv) * d * (4 if dtype == "f32" else 2))
        batch = size(1, 96)
        rows = rng.choice([1, size(1, max(1, min(8192, tokens // batch)))])
        return dict(op=op, batch=batch, rows=rows, ctx=max(rows, size(1, 4096)), nq=nq, nkv=nkv, d=d, page=page,
                    norm=rng.random() < 0.6, dtype=dtype)
    if dtype == "bf16" and rng.random() < 0.4:  # prompts
        rows = size(9, 2048)
        ctx = max(rows, size(9, 8192))
        pairs = 2048 * 8192 * 32
        batch = size(1, max(1, min(16, pairs // (rows * ctx * nq))))
    else:               # single tokens, or a few to verify
        batch = size(1, 64)
        rows = rng.choice([1, 1, 1, 2, 5])
        ctx = max(rows, size(1, 65536))
        ctx = max(rows, min(ctx, 64 * 4096 // batch))
        if dtype == "f32":
            ctx = max(rows, min(ctx, 65536 // batch))
    return dict(op=op, batch=batch, rows=rows, ctx=ctx, nq=nq, nkv=nkv, d=d, page=page, dtype=dtype)


def _lengths(case):
    """(context, new rows) of each sequence: the first one's are the case's, the others' are spread below them."""
    got = []
    for b in range(case["batch"]):
        part = 1.0 if b == 0 else 1.0 - 0.8 * ((b * 37) % 64) / 64
        if case["rows"] == case["ctx"]:  # whole prompts
            rows = max(1, int(case["rows"] * part))
            got.append((rows, rows))
        else:
            rows = case["rows"] if case["rows"] <= 8 else max(1, int(case["rows"] * part))
            got.append((max(rows, int(case["ctx"] * part)), rows))
    return got


# ------------------------------------------------------------------ inputs
def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed * 1000003 + 17)

    def randn(*shape):
        return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32)

    def rand(*shape):
        return torch.rand(*shape, generator=g, device="cuda", dtype=torch.float32)

    dtype = DTYPES[case["dtype"]]
    s = dict(case)
    if case["op"] == "sample":
        rows, vocab = case["rows"], case["vocab"]
        # a few likely tokens over a wide tail, as a language model's logits are
        x = 2.0 * randn(rows, vocab)
        x[:, : vocab // 64] += 6.0 * rand(rows, 1)
        x = x[:, torch.randperm(vocab, generator=g, device="cuda")].contiguous()
        if case["mix"] == "chat":    # one setting for every row
            t = torch.full((rows,), 0.7, device="cuda")
            k = torch.full((rows,), 40, device="cuda", dtype=torch.int32)
            p = torch.full((rows,), 0.95, device="cuda")
            m = torch.full((rows,), 0.0, device="cuda")
        else:                        # each row its own, some of them off, some rows greedy
            t = 0.3 + 1.2 * rand(rows)
            t[rand(rows) < 0.1] = 0.0
            k = (1 + 200 * rand(rows)).to(torch.int32)
            k[rand(rows) < 0.4] = 0
            p = 0.5 + 0.5 * rand(rows)
            p[rand(rows) < 0.3] = 1.0
            m = 0.1 * rand(rows)
            m[rand(rows) < 0.5] = 0.0
        s |= dict(logits=x.to(dtype), uniform=rand(rows), temperature=t, top_k=k, top_p=p, min_p=m)
        return s
    nq, nkv, d, page = case["nq"], case["nkv"], case["d"], case["page"]
    lengths = _lengths(case)
    counts = [(c + page - 1) // page for c, _ in lengths]
    pages, total = max(counts), sum(counts)
    order = torch.randperm(total + 3, generator=g, device="cuda").to(torch.int32)
    table = torch.zeros(len(lengths), pages, dtype=torch.int32)
    order = order.cpu()
    at = 0
    for b, n in enumerate(counts):
        table[b, :n] = order[at:at + n]
        at += n
    starts = [0]
    for _, r in lengths:
        starts.append(starts[-1] + r)
    s |= dict(page_table=table.cuda(), row_start=torch.tensor(starts, dtype=torch.int32, device="cuda"),
              ctx_len=torch.tensor([c for c, _ in lengths], dtype=torch.int32, device="cuda"),
              max_ctx=max(c for c, _ in lengths), max_rows=max(r for _, r in lengths))
    rows = starts[-1]

    def plane():
        """Codes, scales and minima as quantised keys and values have them."""
        scale = 0.3 * (0.8 + 0.4 * rand(total + 3, nkv, page, d // GROUP))
        low = -7.5 * scale + 0.2 * randn(total + 3, nkv, page, d // GROUP)
        code = (7.5 + 3.1 * randn(total + 3, nkv, page, d // 2)).round_().clamp_(0, 15).to(torch.uint8)
        high = (7.5 + 3.1 * randn(total + 3, nkv, page, d // 2)).round_().clamp_(0, 15).to(torch.uint8)
        return code | (high << 4), torch.stack([scale, low], -1).to(torch.float16)

    kc, kp = plane()
    vc, vp = plane()
    s |= dict(cache=(kc, kp, vc, vp))
    if case["op"] == "attend":
        s |= dict(q=(1.5 * randn(rows, nq * d)).to(dtype))
        return s
    pos = torch.arange(s["max_ctx"], device="cuda", dtype=torch.float64)
    freq = 500000.0 ** (-2.0 * torch.arange(d // 2, device="cuda", dtype=torch.float64) / d)
    angle = pos[:, None] * freq
    qkv = randn(rows, (nq + 2 * nkv) * d)
    qkv[:, ::53] *= 4.0   # channels that stand out, as keys have them
    qkv = qkv.to(dtype)   # one projection's output: q, k and v are slices of its rows
    s |= dict(q=qkv[:, : nq * d], k=qkv[:, nq * d: (nq + nkv) * d], v=qkv[:, (nq + nkv) * d:],
              cos_sin=torch.stack([angle.cos(), angle.sin()], -1).float().contiguous(),
              q_norm=(1.0 + 0.1 * randn(d)).to(dtype) if case["norm"] else None,
              k_norm=(1.0 + 0.1 * randn(d)).to(dtype) if case["norm"] else None)
    return s


# ------------------------------------------------------------------ one pass
def run(state):
    if state["op"] == "append":
        return _append_own(state) if own else _append(state)
    if state["op"] == "attend":
        return _attend_own(state) if own else _attend(state)
    return _sample_own(state) if own else _sample(state)


def _append_own(s):
    from aethermind_b200 import ops
    q = ops.kv4_append(s["q"], s["k"], s["v"], s["cache"], s["page_table"], s["row_start"], s["ctx_len"], s["cos_sin"],
                       s["nq"], s["nkv"], s["d"], q_norm=s["q_norm"], k_norm=s["k_norm"], eps=EPS)
    k, v = ops.kv4_gather(s["cache"], s["page_table"], s["row_start"], s["ctx_len"], q.shape[0], s["nkv"], s["d"])
    return {"q": q, "k": k, "v": v}


def _attend_own(s):
    from aethermind_b200 import ops
    return {"out": ops.attention_kv4(s["q"], s["cache"], s["page_table"], s["row_start"], s["ctx_len"], s["nq"],
                                     s["nkv"], s["d"])}


def _sample_own(s):
    from aethermind_b200 import ops
    token, prob = ops.sample(s["logits"], s["uniform"], temperature=s["temperature"], top_k=s["top_k"],
                             top_p=s["top_p"], min_p=s["min_p"], with_prob=True)
    return {"token": token, "prob": prob}


# ------------------------------------------------------------------ the plain forms
def _row_places(s, rows):
    """Sequence and position of every row of the call."""
    r = torch.arange(rows, device="cuda", dtype=torch.int32)
    b = torch.searchsorted(s["row_start"], r, right=True) - 1
    pos = s["ctx_len"][b] - s["row_start"][b + 1] + r
    return b, pos.long()


def _pack(code):
    """Codes [..., d] as a row's bytes [..., d/2]."""
    d = code.shape[-1]
    w = code.to(torch.uint8).unflatten(-1, (d // GROUP, 8, 4, 2)).transpose(-4, -3)
    return (w[..., 0] | (w[..., 1] << 4)).flatten(-3)


def _unpack(codes):
    """A row's bytes [..., d/2] as codes [..., groups, GROUP]."""
    d = 2 * codes.shape[-1]
    w = codes.unflatten(-1, (8, d // GROUP, 4)).transpose(-3, -2)
    return torch.stack([w & 15, w >> 4], -1).flatten(-3)


def _values(codes, params):
    """What rows of the cache stand for, [..., d] in 32 bits."""
    p = params.float()
    return (_unpack(codes).float() * p[..., :1] + p[..., 1:]).flatten(-2)


def _quantise(x):
    """(codes, params) of rows x [..., d] in 32 bits."""
    g = x.unflatten(-1, (-1, GROUP))
    low, high = g.amin(-1), g.amax(-1)
    m = low.clamp(-HALF_MAX, HALF_MAX).to(torch.float16)
    s = ((high - low) / 15.0).clamp(max=STEP_MAX).to(torch.float16)
    sf, mf = s.float()[..., None], m.float()[..., None]
    code = torch.where(sf > 0, ((g - mf) / sf).round().clamp(0, 15), torch.zeros_like(g))
    return _pack(code.flatten(-2)), torch.stack([s, m], -1)


def _norm_rotate(x, weight, cs):
    """x [rows, heads, d] in 32 bits: normalised for each head where there is a weight, then rotated."""
    if weight is not None:
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * weight.float()
    c, sn = cs[:, None, :, 0], cs[:, None, :, 1]
    a, b = x.chunk(2, -1)
    return torch.cat([a * c - b * sn, b * c + a * sn], -1)


def _append(s):
    d, page = s["d"], s["page"]
    rows = s["q"].shape[0]
    b, pos = _row_places(s, rows)
    cs = s["cos_sin"][pos]
    q = _norm_rotate(s["q"].float().unflatten(-1, (-1, d)), s["q_norm"], cs)
    k = _norm_rotate(s["k"].float().unflatten(-1, (-1, d)), s["k_norm"], cs)
    v = s["v"].float().unflatten(-1, (-1, d))
    at, slot = s["page_table"][b, pos // page].long(), pos % page
    kc, kp, vc, vp = s["cache"]
    kc[at, :, slot], kp[at, :, slot] = _quantise(k)
    vc[at, :, slot], vp[at, :, slot] = _quantise(v)
    return {"q": q.flatten(1).to(s["q"].dtype),
            "k": _values(kc[at, :, slot], kp[at, :, slot]).flatten(1).to(torch.bfloat16),
            "v": _values(vc[at, :, slot], vp[at, :, slot]).flatten(1).to(torch.bfloat16)}


def _attend(s):
    nq, nkv, d, page = s["nq"], s["nkv"], s["d"], s["page"]
    batch, n, ctx = s["batch"], s["max_rows"], s["max_ctx"]
    rows = s["q"].shape[0]
    b, pos = _row_places(s, rows)
    place = torch.arange(rows, device="cuda") - s["row_start"][b]
    q = torch.zeros(batch, n, nq, d, device="cuda")
    q[b, place] = s["q"].float().view(rows, nq, d)
    limit = torch.full((batch, n), -1, device="cuda", dtype=torch.long)
    limit[b, place] = pos
    j = torch.arange(ctx, device="cuda")
    at = s["page_table"].long()[:, j // page]                              # [batch, ctx]
    kc, kp, vc, vp = s["cache"]
    k = _values(kc[at, :, j % page], kp[at, :, j % page])                  # [batch, ctx, nkv, d]
    q = q.view(batch, n, nkv, nq // nkv, d).permute(0, 2, 3, 1, 4).reshape(batch, nkv, -1, d)
    score = torch.matmul(q, k.permute(0, 2, 3, 1)).view(batch, nq, n, ctx) * (1.0 / math.sqrt(d))
    del k
    hidden = j > limit[:, None, :, None]
    score.masked_fill_(hidden, -math.inf)
    score -= score.amax(-1, keepdim=True).clamp(min=-1e30)
    score.exp_()
    total = score.sum(-1, keepdim=True)
    v = _values(vc[at, :, j % page], vp[at, :, j % page])
    o = torch.matmul(score.view(batch, nkv, -1, ctx), v.transpose(1, 2)).view(batch, nq, n, d)
    o = o / total.clamp(min=1e-30)
    return {"out": o.transpose(1, 2)[b, place].reshape(rows, nq * d).to(s["q"].dtype)}


def _sample(s):
    x = s["logits"].float()
    x = torch.where(torch.isnan(x), torch.full_like(x, -math.inf), x)
    top = x.amax(-1, keepdim=True)
    greedy = ~(s["temperature"] > 0)
    t = torch.where(greedy, torch.ones_like(s["temperature"]), s["temperature"])
    z = torch.where(x == top, torch.zeros_like(x), (x - top) / t[:, None])
    z, order = torch.sort(z, dim=-1, descending=True, stable=True)
    w = (torch.exp(z) * ONE).long()
    rank = torch.arange(x.shape[1], device="cuda")
    least = torch.where(s["min_p"] > 0, s["min_p"].double() * ONE, torch.zeros_like(s["min_p"].double())).ceil().long()
    k = torch.where(s["top_k"] > 0, s["top_k"].long(), torch.full_like(s["top_k"].long(), x.shape[1]))
    k = torch.where(greedy, torch.ones_like(k), k)
    w = torch.where((w >= least[:, None]) & (rank < k[:, None]), w, torch.zeros_like(w))
    before = w.cumsum(-1) - w
    want = torch.where(s["top_p"] < 1, (s["top_p"].double() * w.sum(-1).double()).ceil().long(), w.sum(-1))
    w = torch.where((before < want[:, None]) | (rank == 0), w, torch.zeros_like(w))
    total = w.sum(-1)
    w = torch.zeros_like(w).scatter_(1, order, w)                           # back in the order of the vocabulary
    r = torch.minimum((s["uniform"].double() * total.double()).floor().long(), total - 1)
    token = (w.cumsum(-1) > r[:, None]).to(torch.uint8).argmax(-1)
    prob = w.gather(1, token[:, None])[:, 0].float() / total.float()
    none = top[:, 0] == -math.inf
    return {"token": torch.where(none, torch.full_like(token, -1), token),
            "prob": torch.where(none, torch.zeros_like(prob), prob)}


# ------------------------------------------------------------------ in 64 bits, from the definitions
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "append":
        return _append_exact(s)
    if case["op"] == "attend":
        return _attend_exact(s)
    return _sample_exact(s)


def _row_exact(codes, params):
    """Rows of bytes as values, nibble by nibble."""
    d = 2 * codes.shape[-1]
    groups = d // GROUP
    out = torch.empty(*codes.shape[:-1], d, dtype=torch.float64, device=codes.device)
    for e in range(d):
        g, i = divmod(e, GROUP)
        byte = 4 * ((i // 8) * groups + g) + (i % 8) // 2
        c = (codes[..., byte] >> (4 * (i % 2))) & 15
        out[..., e] = params[..., g, 0].double() * c.double() + params[..., g, 1].double()
    return out


def _sequences(s):
    starts, ctxs, table = s["row_start"].tolist(), s["ctx_len"].tolist(), s["page_table"].long()
    for b, ctx in enumerate(ctxs):
        yield slice(starts[b], starts[b + 1]), ctx, table[b]


def _append_exact(s):
    d = s["d"]

    def turned(x, weight, pos):
        x = x.double().view(x.shape[0], -1, d)
        if weight is not None:
            x = x / (x.square().mean(-1, keepdim=True) + EPS).sqrt() * weight.double()
        cs = s["cos_sin"][pos].double()
        a, b = x[..., : d // 2], x[..., d // 2:]
        c, sn = cs[:, None, :, 0], cs[:, None, :, 1]
        return torch.cat([a * c - b * sn, a * sn + b * c], -1)

    def held(x):
        g = x.view(x.shape[0], -1, d // GROUP, GROUP)
        m = g.amin(-1, keepdim=True).to(torch.float16).double()
        step = ((g.amax(-1, keepdim=True) - g.amin(-1, keepdim=True)) / 15).to(torch.float16).double()
        code = torch.where(step > 0, ((g - m) / step.clamp(min=1e-12)).round().clamp(0, 15), torch.zeros_like(g))
        return (code * step + m).reshape(x.shape[0], -1)

    q, k, v = [], [], []
    for at, ctx, _ in _sequences(s):
        pos = torch.arange(ctx - (at.stop - at.start), ctx, device="cuda")
        q.append(turned(s["q"][at], s["q_norm"], pos).flatten(1))
        k.append(held(turned(s["k"][at], s["k_norm"], pos)))
        v.append(held(s["v"][at].double().view(-1, s["nkv"], d)))
    return {"q": torch.cat(q), "k": torch.cat(k), "v": torch.cat(v)}


def _attend_exact(s):
    nq, nkv, d, page = s["nq"], s["nkv"], s["d"], s["page"]
    kc, kp, vc, vp = s["cache"]
    out = torch.zeros(s["q"].shape[0], nq * d, dtype=torch.float64, device="cuda")
    for at, ctx, table in _sequences(s):
        n = at.stop - at.start
        used = table[: (ctx + page - 1) // page]
        seen = torch.arange(ctx, device="cuda")[None, :] <= torch.arange(ctx - n, ctx, device="cuda")[:, None]
        for h in range(nkv):
            k = _row_exact(kc[used, h].flatten(0, 1)[:ctx], kp[used, h].flatten(0, 1)[:ctx])
            v = _row_exact(vc[used, h].flatten(0, 1)[:ctx], vp[used, h].flatten(0, 1)[:ctx])
            for i in range(h * (nq // nkv), (h + 1) * (nq // nkv)):
                score = s["q"][at, i * d:(i + 1) * d].double() @ k.T / math.sqrt(d)
                score = torch.where(seen, score, -math.inf)
                out[at, i * d:(i + 1) * d] = torch.softmax(score, -1) @ v
    return {"out": out}


def _sample_exact(s):
    """The chosen token's probability; the token itself hangs on the roundings that the definition names."""
    prob = []
    for i in range(s["logits"].shape[0]):
        x = s["logits"][i].double()
        t = float(s["temperature"][i])
        if not t > 0:
            prob.append(1.0)
            continue
        p, order = torch.sort(torch.softmax(x / t, -1), descending=True, stable=True)
        keep = torch.ones_like(p, dtype=torch.bool)
        if s["min_p"][i] > 0:
            keep &= p >= s["min_p"][i].double() * p[0]
        if s["top_k"][i] > 0:
            keep[int(s["top_k"][i]):] = False
        p = torch.where(keep, p, 0.0)
        if s["top_p"][i] < 1:
            before = p.cumsum(-1) - p
            p = torch.where(before < s["top_p"][i].double() * p.sum(), p, 0.0)
        p = torch.zeros_like(p).scatter_(0, order, p / p.sum())
        run_ = p.cumsum(-1)
        u = s["uniform"][i].double()
        if (run_ - u).abs().min() < 1e-8:  # a draw on the border of two tokens: 64 bits may name the other one
            return {"token": None, "prob": None}
        prob.append(float(p[int((run_ > u).to(torch.uint8).argmax())]))
    return {"token": None, "prob": torch.tensor(prob, dtype=torch.float64)}


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    size = 4 if case["dtype"] == "f32" else 2
    if case["op"] == "sample":
        n = case["rows"] * case["vocab"]
        return {"bytes": n * size + case["rows"] * 32, "flops": 4 * n}
    nq, nkv, d = case["nq"], case["nkv"], case["d"]
    lengths = _lengths(case)
    rows = sum(r for _, r in lengths)
    token = 2 * nkv * (d // 2 + 4 * (d // GROUP))  # a token's keys and values in the cache
    if case["op"] == "append":
        values = 2 * rows * nkv * d * 2            # read back as bf16
        return {"bytes": rows * (2 * nq + 2 * nkv) * d * size + rows * token + values + rows * d * 4,
                "flops": rows * (10 * nq + 20 * nkv) * d}
    pairs = sum(r * c - r * (r - 1) // 2 for c, r in lengths)
    return {"bytes": sum(c for c, _ in lengths) * token + 2 * rows * nq * d * size, "flops": 4 * pairs * nq * d}
