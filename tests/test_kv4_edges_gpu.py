"""The 4-bit paged KV cache where calls go wrong: positions that do not exist, numbers that are none, rows of which one
token has nearly all the mass, and calls large enough for the kernels of prompts."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

import kv4_reference as ref  # noqa: E402
import test_kv4_gpu as base  # noqa: E402
from test_kv4_gpu import bf16, check_attention, dev, di, make_batch, poison_unused, random_cache  # noqa: E402

pytestmark = pytest.mark.gpu

OUT_OF_RANGE = 11


@pytest.fixture(scope="module")
def ops(built_lib):
    from aethermind_b200 import ops as O
    return O


def i32(a):
    return torch.tensor(a, dtype=torch.int32, device="cuda")


# ------------------------------------------------------------------ the status word
@pytest.mark.parametrize("n,keys,nq,nkv,d", [
    (700, 60, 12, 1, 64),   # each warp takes whole items
    (128, 96, 32, 8, 128),
    (5, 60, 12, 1, 64),     # shares of all units
])
def test_attention_reports_a_context_past_the_page_table(ops, n, keys, nq, nkv, d):
    """Whichever of many sequences it is, and nothing where there is none."""
    rng = np.random.default_rng(n)
    pages = -(-keys // 16)
    table, start, ctx, total = make_batch([(keys, 1)] * n, 16, rng, pages=pages)
    cache = dev(random_cache(total, nkv, 16, d, rng))
    q = bf16(rng.normal(0, 1, (n, nq * d))).cuda()
    wrong = []
    for at in [None, *range(n)]:
        c = ctx.copy()
        if at is not None:
            c[at] = pages * 16 + 5
        status = i32([0])
        ops.attention_kv4(q, cache, di(table), di(start), di(c), nq, nkv, d, status=status)
        if status.item() != (0 if at is None else OUT_OF_RANGE):
            wrong.append(at)
    assert not wrong


@pytest.mark.parametrize("lens,nq,nkv,d", [
    ([(2, 3)], 8, 2, 64),
    ([(300, 1), (2, 3)], 8, 2, 64),
    ([(20, 1)] * 150 + [(2, 3)] + [(20, 1)] * 30, 32, 8, 64),
    ([(300, 160), (20, 21)], 32, 8, 128),  # the kernel of prompts
    ([(0, 160)], 32, 8, 64),
])
@pytest.mark.parametrize("short", [True, False])
def test_attention_reports_rows_before_position_0(ops, lens, nq, nkv, d, short):
    """A context below its rows is reported, as kv4_append does; as many keys as rows are not."""
    rng = np.random.default_rng(2)
    lens = lens if short else [(max(c, n), n) for c, n in lens]
    table, start, ctx, total = make_batch(lens, 16, rng)
    cache = dev(random_cache(total, nkv, 16, d, rng))
    q = bf16(rng.normal(0, 1, (start[-1], nq * d))).cuda()
    status = i32([0])
    ops.attention_kv4(q, cache, di(table), di(start), di(ctx), nq, nkv, d, status=status)
    assert status.item() == (OUT_OF_RANGE if short else 0)


# ------------------------------------------------------------------ numbers that are none
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("lens,nq,nkv,d", [
    ([(5, 1), (40, 3)], 8, 2, 128),
    ([(9000, 2)], 8, 2, 64),               # items cut between CTAs
    ([(30, 1)] * 160, 32, 8, 128),         # each warp takes whole items
    ([(20, 21), (300, 160)], 32, 8, 128),  # bf16: the kernel of prompts; the first row sees no key
    ([(400, 190)], 32, 8, 64),
])
def test_attention_of_a_q_that_is_no_number(ops, lens, nq, nkv, d, bad, dtype):
    """The row's head is NaN where it sees a key, 0 where it sees none; every other head is as it would be."""
    rng = np.random.default_rng(3)
    table, start, ctx, total = make_batch(lens, 16, rng)
    cache = random_cache(total, nkv, 16, d, rng)
    cache[1][..., 1] = 0.25  # all keys above zero: an infinite element gives scores of one sign
    poison_unused(cache, table, ctx)
    rows = start[-1]
    q = torch.from_numpy(rng.normal(0, 1.5, (rows, nq * d)).astype(np.float32)).to(dtype)
    want = ref.attention(q.double().numpy(), cache, table, start, ctx, nq, nkv, d)
    hit = [(0, 1, 3), (rows - 1, nq - 1, d - 1), (rows // 2, 2, d // 2)]
    for r, h, e in hit:
        q[r, h * d + e] = bad
    got = ops.attention_kv4(q.cuda(), dev(cache), di(table), di(start), di(ctx), nq, nkv, d)
    b = np.repeat(np.arange(len(lens)), np.diff(start))
    for r, h, _ in hit:
        part = got[r, h * d:(h + 1) * d]
        if ctx[b[r]] - start[b[r] + 1] + r >= 0:
            assert torch.isnan(part).all(), (r, h)
        else:
            assert (part == 0).all(), (r, h)
        part.copy_(torch.from_numpy(want[r, h * d:(h + 1) * d]))
    check_attention(got, want, dtype, 4.0)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("steps", [1, 4])
def test_append_of_groups_that_are_no_numbers(ops, d, steps, dtype):
    """A group of NaN alone reads as NaN, whether a norm made it or not; its neighbours are as they would be."""
    rng = np.random.default_rng(7)
    nq, nkv, page = 8, 2, 32
    rows = 24 if steps == 1 else 7000  # few and many steps to a warp
    x = torch.from_numpy(rng.normal(0, 1, (rows, (nq + 2 * nkv) * d)).astype(np.float32)).to(dtype).cuda()
    k0, v0 = nq * d, (nq + nkv) * d
    bad = x.clone()
    bad[3, v0: v0 + 64] = float("nan")            # the first group of a value
    bad[5, v0 + 2 * d - 64: v0 + 2 * d] = float("nan")   # the last one of the row
    bad[9, k0 + d + 7] = float("nan")             # one element of a key: the norm spreads it over the head
    cs = torch.from_numpy(ref.rope_table(10000.0, d, rows)).cuda()
    pages = -(-rows // page)
    args = (i32([list(range(pages))]), i32([0, rows]), i32([rows]))
    w = torch.ones(d, dtype=dtype, device="cuda")
    got = []
    for t in (x, bad):
        cache = ops.kv4_cache(pages, page, nkv, d)
        q = ops.kv4_append(t[:, :k0], t[:, k0:v0], t[:, v0:], cache, *args, cs, nq, nkv, d, q_norm=w, k_norm=w)
        got.append((q, *ops.kv4_gather(cache, *args, rows, nkv, d, dtype=torch.float32)))
    (q, k, v), (bq, bk, bv) = got
    assert torch.equal(q, bq)
    assert torch.isnan(bk[9, d:]).all()
    bk[9, d:] = k[9, d:]
    assert torch.isnan(bv[3, :64]).all() and torch.isnan(bv[5, -64:]).all()
    bv[3, :64], bv[5, -64:] = v[3, :64], v[5, -64:]
    assert torch.equal(k, bk) and torch.equal(v, bv)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("pair", [(0, np.nan), (np.nan, 0.5)])  # scale and minimum of a group that is no number
@pytest.mark.parametrize("lens,at,nq,nkv,d", [
    ([(40, 5), (40, 5)], 37, 8, 2, 128),   # rows 0 and 1 of five do not see it
    ([(40, 5), (40, 5)], 3, 8, 2, 64),
    ([(9000, 3)], 8998, 8, 2, 64),         # items cut between CTAs
    ([(9000, 3)], 4001, 8, 2, 128),
    ([(30, 2)] * 160, 29, 32, 8, 128),     # each warp takes whole items
    ([(300, 160)], 220, 32, 8, 128),       # bf16: the kernel of prompts
    ([(400, 190), (300, 20)], 399, 32, 8, 64),
    ([(300, 160)], 5, 32, 8, 128),
])
def test_attention_over_keys_and_values_that_are_no_numbers(ops, lens, at, nq, nkv, d, pair, dtype):
    """A NaN key is in every element of the rows that see it, a NaN group of a value in its 64 elements of them, and
    neither is in another row, head or sequence."""
    rng = np.random.default_rng(11)
    table, start, ctx, total = make_batch(lens, 16, rng)
    cache = random_cache(total, nkv, 16, d, rng)
    poison_unused(cache, table, ctx)
    rows = start[-1]
    q = torch.from_numpy(rng.normal(0, 1.5, (rows, nq * d)).astype(np.float32)).to(dtype)
    want = ref.attention(q.double().numpy(), cache, table, start, ctx, nq, nkv, d)
    heads, grp = want.reshape(rows, nq, d).copy(), nq // nkv
    kc, kp, vc, vp = cache
    for b, (kh, vh, g) in ((0, (0, 1, 0)), (len(lens) - 1, (1, 0, d // 64 - 1))):
        if at >= ctx[b]:
            continue
        page, slot = table[b, at // 16], at % 16
        for par, h, i in ((kp, kh, 0), (vp, vh, g)):
            par[page, h, slot, i] = pair
        for r in range(start[b], start[b + 1]):
            if ctx[b] - start[b + 1] + r >= at:
                heads[r, kh * grp:(kh + 1) * grp] = np.nan
                heads[r, vh * grp:(vh + 1) * grp, 64 * g:64 * g + 64] = np.nan
    got = ops.attention_kv4(q.cuda(), dev(cache), di(table), di(start), di(ctx), nq, nkv, d)
    nan = torch.from_numpy(np.isnan(heads).reshape(rows, -1)).cuda()
    assert nan.any() and torch.equal(torch.isnan(got), nan)
    got[nan] = torch.from_numpy(want).to(dtype).cuda()[nan]
    check_attention(got, want, dtype, 4.0)


# ------------------------------------------------------------------ numbers far apart
@pytest.mark.parametrize("s", [6e-8, 1e-6, 1e-4])
@pytest.mark.parametrize("hole", [False, True])
@pytest.mark.parametrize("n", [1, 150])
def test_attention_small_values_after_zeros(ops, s, hole, n):
    """Values of one number only (scale 0), or a page that is none, before values with the smallest scales. bf16:
    p and p s are rounded to 11 bits, the result to 8: 2^-8 of its norm."""
    rng = np.random.default_rng(4)
    nq, nkv, d = 8, 2, 128
    table, start, ctx, total = make_batch([(400, 1)] * n, 16, rng)
    cache = random_cache(total, nkv, 16, d, rng)
    cache[3][..., 0] = np.float16(s)
    cache[3][..., 1] = 0
    cache[3][table[:, :9], ..., 0] = 0
    if hole:
        table[:, 0] = -1
    q = bf16(rng.normal(0, 1, (n, nq * d)))
    want = ref.attention(q.double().numpy(), cache, table, start, ctx, nq, nkv, d)
    got = ops.attention_kv4(q.cuda(), dev(cache), di(table), di(start), di(ctx), nq, nkv, d).double().cpu().numpy()
    assert np.linalg.norm(got - want) <= 2.0 ** -8 * np.linalg.norm(want)


def one_token_with_most_of_the_mass(lens, nq, nkv, d, dtype, s, s_first):
    """Inputs whose first key is e^3 to e^14 times as likely as every other one (by row and head), and the result.
    s: V's scale (its minimum is 0), s_first: the first key's. All other keys are alike, so that a rounding of p or of
    p s is every key's and does not average out."""
    rng = np.random.default_rng(5)
    page = 64
    table, start, ctx, total = make_batch(lens, page, rng)
    kc, kp, vc, vp = random_cache(total, nkv, page, d, rng)
    kp[..., 0], kp[..., 1] = 0, 0.25
    vp[..., 0], vp[..., 1] = np.float16(s), 0
    kp[table[:, 0], :, 0, :, 1] = 1.25
    vp[table[:, 0], :, 0, :, 0] = np.float16(s_first)
    rows = start[-1]
    gap = np.linspace(3, 14, rows * nq).reshape(rows, nq)
    q = torch.from_numpy(np.repeat(gap / d, d, 1).astype(np.float32)).to(dtype)
    rest = np.exp(-q.double().numpy().reshape(rows, nq, d).sum(-1))  # the others' p
    want = np.zeros((rows, nq, d))
    for b, (c, n) in enumerate(lens):
        v = ref.values(vc[table[b]], vp[table[b]]).transpose(1, 0, 2, 3).reshape(nkv, -1, d)
        total_v = np.cumsum(v[:, 1:], 1)
        for r in range(start[b], start[b + 1]):
            others = c - n + r - start[b]
            for h in range(nq):
                e, g = rest[r, h], h // (nq // nkv)
                want[r, h] = (v[g, 0] + e * total_v[g, others - 1]) / (1 + e * others)
    return (q.cuda(), dev((kc, kp, vc, vp)), di(table), di(start), di(ctx), nq, nkv, d), want


def worst_head(got, want):
    got = got.double().cpu().numpy().reshape(want.shape)
    return (np.linalg.norm(got - want, axis=-1) / np.linalg.norm(want, axis=-1)).max()


@pytest.mark.parametrize("s,s_first", [(0.3, 0), (0.07, 0), (0.04, 0), (3.0, 0), (9.0, 0), (100.0, 0), (0.3, 0.3),
                                       (0.3, 30.0), (100.0, 0.3), (1e-5, 4000.0)])
@pytest.mark.parametrize("lens,nq,nkv,d", [
    ([(600, 1)] * 160, 32, 8, 64),   # each warp takes whole items
    ([(20000, 1)], 12, 2, 128),      # items cut between CTAs
    ([(300, 2), (90, 1)], 8, 2, 128),
])
def test_attention_of_one_token_with_most_of_the_mass(ops, lens, nq, nkv, d, s, s_first):
    """bf16: p and p s are rounded to 11 bits (2^-12 each), the result to 8 (2^-9): no head is off by 2^-8."""
    args, want = one_token_with_most_of_the_mass(lens, nq, nkv, d, torch.bfloat16, s, s_first)
    assert worst_head(ops.attention_kv4(*args, scale=1.0), want) <= 2.0 ** -8


def in_the_kernel_of_prompts(lens, nq, nkv, sms=148):
    """The rule by which bf16 calls go to the kernel of prompts."""
    cols = sum(n for _, n in lens) * (nq // nkv)
    tiles = (cols // 256 + len(lens)) * nkv
    return -(-cols // 8) * nkv * 2 > 5 * sms * -(-tiles // sms)


@pytest.mark.parametrize("s_first", [0, 0.3, 30.0])
@pytest.mark.parametrize("lens,nq,nkv,d", [([(8192, 200)], 16, 1, 64), ([(8192, 200)], 16, 1, 128),
                                           ([(4000, 160), (700, 100)], 32, 8, 64)])
def test_attention_prompts_of_one_token_with_most_of_the_mass(ops, lens, nq, nkv, d, s_first):
    """As above; p is rounded once (2^-12), the result to 8 bits (2^-9)."""
    assert in_the_kernel_of_prompts(lens, nq, nkv)
    args, want = one_token_with_most_of_the_mass(lens, nq, nkv, d, torch.bfloat16, 0.3, s_first)
    assert worst_head(ops.attention_kv4(*args, scale=1.0), want) <= 2.0 ** -8


@pytest.mark.parametrize("s,s_first", [(0.3, 0), (0.04, 0), (100.0, 0), (0.3, 30.0), (100.0, 0.3)])
@pytest.mark.parametrize("lens,nq,nkv,d", [([(600, 1)] * 160, 32, 8, 64), ([(20000, 1)], 12, 2, 128),
                                           ([(300, 2), (90, 1)], 8, 2, 128)])
def test_attention_fp32_of_one_token_with_most_of_the_mass(ops, lens, nq, nkv, d, s, s_first):
    """fp32: a score of up to 14 carries an error of 2^-20 from its fp32 sums, p and the elements of V 2^-22 each: below
    4e-6 in all."""
    args, want = one_token_with_most_of_the_mass(lens, nq, nkv, d, torch.float32, s, s_first)
    assert worst_head(ops.attention_kv4(*args, scale=1.0), want) <= 4e-6


# ------------------------------------------------------------------ rows that are nowhere
@pytest.mark.parametrize("d,many", [(64, False), (64, True), (128, True)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_append_rows_out_of_range_give_zeros(ops, d, many, dtype):
    """q_out of rows before position 0 or past the rotation table is zero, in both layouts of the kernel."""
    rng = np.random.default_rng(4)
    nq, nkv, page = 6, 1, 16
    n = 12000 if many else 0  # further rows, so that a warp takes several steps
    table = np.arange(3 * 800, dtype=np.int32).reshape(3, 800)
    start, ctx = np.array([0, 4, 8, 8 + n], np.int32), np.array([18, 2, n], np.int32)
    rows = 8 + n
    x = torch.from_numpy(rng.normal(0, 1, (rows, (nq + 2) * d)).astype(np.float32)).to(dtype).cuda()
    cs = torch.from_numpy(ref.rope_table(10000.0, d, max(n, 17))).cuda()  # position 17 of sequence 0 where n is 0
    cache = ops.kv4_cache(3 * 800, page, nkv, d)
    status = i32([0])
    args = (x[:, nq * d: (nq + 1) * d], x[:, (nq + 1) * d:], cache, di(table), di(start), di(ctx), cs, nq, nkv, d)
    out = torch.full((rows, nq * d), float("nan"), dtype=dtype, device="cuda")
    ops.kv4_append(x[:, : nq * d], *args, q_out=out, status=status)
    zero = (out == 0).all(1).cpu().numpy()
    want = np.zeros(rows, bool)
    want[4:6] = True          # positions -2, -1
    want[3] = not many        # position 17, past the table
    np.testing.assert_array_equal(zero, want)
    assert not torch.isnan(out).any() and status.item() == OUT_OF_RANGE


@pytest.mark.parametrize("starts", [[0, 2, 4], [1, 2, 6], [2, 3, 4], [0, 0, 0], [6, 6, 6]])
def test_append_and_gather_rows_of_no_sequence(ops, starts):
    d, nq, nkv = 64, 4, 2
    x = torch.ones(6, 8 * d, dtype=torch.bfloat16, device="cuda")
    cs = torch.from_numpy(ref.rope_table(10000.0, d, 64)).cuda()
    args = (i32([[0], [1]]), i32(starts), i32([9, 9]))
    none = torch.tensor([not starts[0] <= r < starts[-1] for r in range(6)])
    cache, status = ops.kv4_cache(2, 16, nkv, d), i32([0])
    out = torch.full((6, nq * d), float("nan"), dtype=torch.bfloat16, device="cuda")
    ops.kv4_append(x[:, : nq * d], x[:, : nkv * d], x[:, : nkv * d], cache, *args, cs, nq, nkv, d, q_out=out,
                   status=status)
    assert torch.equal((out == 0).all(1).cpu(), none) and status.item() == OUT_OF_RANGE
    status.zero_()
    k, v = ops.kv4_gather(cache, *args, 6, nkv, d, status=status)
    assert torch.equal((k == 0).all(1).cpu(), none) and torch.equal((v == 0).all(1).cpu(), none)
    assert status.item() == OUT_OF_RANGE


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,starts,lens", [
    (6, [0, 2, 4], [9, 9]), (6, [1, 2, 6], [9, 9]), (6, [2, 3, 4], [9, 9]), (6, [0, 0, 0], [9, 9]),
    (400, list(range(5, 396)), [20] * 390),     # each warp takes whole items
    (300, [3, 180, 290], [300, 200]),                 # bf16: the kernel of prompts
    (700, [0, 0, 0], [300, 200]),
])
def test_attention_rows_of_no_sequence(ops, rows, starts, lens, dtype):
    """They are zero and reported; the others are as in a call without them."""
    rng = np.random.default_rng(6)
    nq, nkv, d = 32, 8, 64
    pages = -(-max(lens) // 16)
    cache = dev(random_cache(pages * len(lens), nkv, 16, d, rng))
    table = i32(np.arange(pages * len(lens)).reshape(len(lens), pages).tolist())
    q = torch.from_numpy(rng.normal(0, 1, (rows, nq * d)).astype(np.float32)).to(dtype).cuda()
    status = i32([0])
    out = torch.full((rows, nq * d), float("nan"), dtype=dtype, device="cuda")
    ops.attention_kv4(q, cache, table, i32(starts), i32(lens), nq, nkv, d, out=out, status=status)
    first, end = starts[0], starts[-1]
    assert (out[:first] == 0).all() and (out[end:] == 0).all() and status.item() == OUT_OF_RANGE
    if end > first:
        status.zero_()
        alone = ops.attention_kv4(q[first:end].clone(), cache, table, i32([x - first for x in starts]), i32(lens), nq,
                                  nkv, d, status=status)
        assert status.item() == 0
        err = (out[first:end].double() - alone.double()).norm() / alone.double().norm()
        assert err <= (2.0 ** -8 if dtype == torch.bfloat16 else 1e-5)


def test_rows_but_no_sequence(ops):
    d, nq, nkv, rows = 64, 4, 2, 5
    cache, status = ops.kv4_cache(2, 16, nkv, d), i32([0])
    x = torch.ones(rows, nq * d, dtype=torch.bfloat16, device="cuda")
    cs = torch.from_numpy(ref.rope_table(10000.0, d, 64)).cuda()
    args = (cache, torch.zeros(0, 1, dtype=torch.int32, device="cuda"), i32([0]), i32([]))

    def out():
        return torch.full((rows, nq * d), float("nan"), dtype=torch.bfloat16, device="cuda")

    for call in (lambda: [ops.attention_kv4(x, *args, nq, nkv, d, out=out(), status=status)],
                 lambda: ops.kv4_gather(*args, rows, nkv, d, status=status),
                 lambda: [ops.kv4_append(x, x[:, : nkv * d], x[:, : nkv * d], *args, cs, nq, nkv, d, q_out=out(),
                                         status=status)]):
        status.zero_()
        torch.empty(rows, nq * d, dtype=torch.bfloat16, device="cuda").fill_(float("nan"))  # what fresh memory may hold
        assert all((t == 0).all() for t in call()) and status.item() == OUT_OF_RANGE


# ------------------------------------------------------------------ calls that are large enough for other layouts
@pytest.mark.parametrize("norms", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("lens,nq,nkv,d,page", [
    ([(2100, 2100), (1000, 700), (3, 1), (0, 0), (4000, 3900)], 32, 8, 64, 64),
    ([(2500, 2500), (900, 77)], 13, 3, 128, 16),             # heads that do not fill a warp's steps
    ([(9000, 8900), (700, 699), (1, 1)], 5, 1, 64, 256),
    ([(5000, 4900)], 7, 1, 128, 32),
])
def test_append_of_prompts(ops, lens, nq, nkv, d, page, dtype, norms):
    """The kernel that takes four steps to a warp (rows times steps above 128 an SM), bit for bit without norms."""
    assert sum(n for _, n in lens) * -(-(nq + 2 * nkv) // (256 // d)) > 128 * 148
    (base.test_append_with_norms if norms else base.test_append_bit_exact_without_norm)(ops, lens, nq, nkv, d, page, dtype)


def rising(lens, nq, nkv, d, exact):
    """A cache whose scores grow by hundreds along the keys. exact: every key is a whole number of 2^-4 below 2^7, so
    that 11 bits hold it."""
    rng = np.random.default_rng(31)
    page = 64
    table, start, ctx, total = make_batch(lens, page, rng)
    kc, kp, vc, vp = random_cache(total, nkv, page, d, rng)
    if exact:
        kp[..., 0], kp[..., 1] = 2.0 ** -4, -0.5
    for b, (c, _) in enumerate(lens):
        for i in range(c):
            step = np.round(0.16 * i) / 16 if exact else 0.01 * i
            kp[table[b, i // page], :, i % page, :, 1] += np.float16(step)
    q = bf16(np.abs(rng.normal(0, 1, (start[-1], nq * d))))
    want = ref.attention(q.double().numpy(), (kc, kp, vc, vp), table, start, ctx, nq, nkv, d)
    return (q.cuda(), dev((kc, kp, vc, vp)), di(table), di(start), di(ctx), nq, nkv, d), want


@pytest.mark.parametrize("lens,nq,nkv,d", [([(700, 150)], 32, 8, 128), ([(700, 200), (300, 60)], 32, 8, 64),
                                           ([(520, 130)], 40, 8, 128)])
def test_attention_prompts_of_rising_scores(ops, lens, nq, nkv, d):
    """The softmax reference moves many times in the kernel of prompts. Scores of hundreds in fp32 sums: 2^-13 in the
    exponent; p to 11 bits and the result to 8: 2^-8."""
    assert in_the_kernel_of_prompts(lens, nq, nkv)
    args, want = rising(lens, nq, nkv, d, exact=True)
    got = ops.attention_kv4(*args).double().cpu().numpy()
    assert np.linalg.norm(got - want) <= 2.0 ** -8 * np.linalg.norm(want)


@pytest.mark.parametrize("exact", [True, False])
@pytest.mark.parametrize("lens,nq,nkv,d", [([(700, 64)], 32, 8, 128), ([(700, 3), (90, 1)], 32, 8, 64)])
def test_attention_of_rising_scores(ops, lens, nq, nkv, d, exact):
    """The same in the kernel of single tokens, whose codes are exact whatever the scale: sums of hundreds to 2^-17 of
    their largest term are 2^-8 in the exponent, the result 2^-9."""
    assert not in_the_kernel_of_prompts(lens, nq, nkv)
    args, want = rising(lens, nq, nkv, d, exact)
    got = ops.attention_kv4(*args).double().cpu().numpy()
    assert np.linalg.norm(got - want) <= 2.0 ** -7 * np.linalg.norm(want)


@pytest.mark.parametrize("lens,nq,nkv,d,page", [
    ([(200, 130)], 32, 8, 128, 64),
    ([(129, 95), (300, 64), (3, 1), (0, 0), (257, 63)], 32, 8, 128, 32),
    ([(200, 100), (383, 33)], 64, 8, 128, 16),
    ([(485, 229), (90, 2)], 32, 8, 64, 256),
    ([(513, 300)], 16, 16, 64, 128),
    ([(3000, 3000)], 1, 1, 64, 32),     # one q head to a kv head
    ([(400, 400)], 24, 3, 128, 16),
])
def test_attention_in_the_kernel_of_prompts(ops, lens, nq, nkv, d, page):
    assert in_the_kernel_of_prompts(lens, nq, nkv)
    base.test_attention_prompts(ops, lens, nq, nkv, d, page)
