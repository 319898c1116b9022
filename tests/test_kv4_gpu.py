"""The 4-bit paged KV cache on the GPU against a plain 64-bit implementation.

Tolerances, from the arithmetic:
* bf16 outputs: half an ulp is 2^-9 of a value; with p and v rounded to 11 bits on the way (2^-11 each of the largest
  |v|) the error's norm stays below 2^-8 of the result's, and no element is off by more than 2^-8 |y| + 2^-9 max |v|.
* fp32 outputs: products to 22 bits, sums in 32: scores of a few tens carry an absolute error of some 2^-19, so the
  norm's error stays below 1e-5.
* codes: with the rotation's products rounded one by one in fp32, the codes and parameters of rows without a norm are
  equal bit for bit to the same expressions in numpy float32; with a norm (another order of the sum of squares) a code
  may differ by one where the quotient is within 2^-8 of a half, and a parameter by one fp16 ulp.
"""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

import kv4_reference as ref  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops(built_lib):
    from aethermind_b200 import ops as O
    return O


def bf16(a):
    return torch.from_numpy(np.ascontiguousarray(a, np.float32)).to(torch.bfloat16)


def make_batch(lens, page, rng, spare=2, pages=None):
    """lens: (ctx, new rows) per sequence -> page_table, row_start, ctx_len (numpy), number of pages."""
    counts = [-(-max(c, 0) // page) for c, _ in lens]
    total = sum(counts) + spare
    order = rng.permutation(total).astype(np.int32)
    width = max(counts + [1]) if pages is None else pages
    table = np.full((len(lens), width), -7, np.int32)  # unused entries are no pages
    at = 0
    for b, n in enumerate(counts):
        table[b, :n] = order[at:at + n]
        at += n
    start = np.concatenate([[0], np.cumsum([n for _, n in lens])]).astype(np.int32)
    return table, start, np.array([c for c, _ in lens], np.int32), total


def random_cache(total, nkv, page, d, rng, poison=True):
    """A full cache; every byte of it is defined, also where no token is (NaN and inf parameters there)."""
    def plane():
        codes = rng.integers(0, 256, (total, nkv, page, d // 2), dtype=np.uint8)
        s = rng.uniform(0.05, 0.4, (total, nkv, page, d // 64)).astype(np.float16)
        m = (-7.5 * s + rng.normal(0, 0.3, s.shape)).astype(np.float16)
        return codes, np.stack([s, m], -1)
    return (*plane(), *plane())


def poison_unused(cache, table, ctx_len):
    """NaN / inf parameters wherever no visible token is."""
    kc, kp, vc, vp = cache
    page = kc.shape[2]
    used = np.zeros((kc.shape[0], page), bool)
    for b, c in enumerate(ctx_len):
        for p in range(max(0, c)):
            if p // page < table.shape[1] and 0 <= table[b, p // page] < kc.shape[0]:
                used[table[b, p // page], p % page] = True
    for par, bad in ((kp, np.nan), (vp, np.inf)):
        np.moveaxis(par, 2, 1)[~used] = bad


def dev(cache):
    return tuple(torch.from_numpy(np.ascontiguousarray(c)).cuda() for c in cache)


def di(a):
    return torch.from_numpy(a).cuda()


def check_attention(got, want, dtype, vmax):
    got = got.double().cpu().numpy()
    assert np.isfinite(got).all()
    norm = np.linalg.norm(want)
    err = np.linalg.norm(got - want)
    if dtype == torch.bfloat16:
        assert err <= 2.0 ** -8 * norm + 1e-30, err / max(norm, 1e-30)
        assert (np.abs(got - want) <= 2.0 ** -8 * np.abs(want) + 2.0 ** -9 * vmax).all()
    else:
        assert err <= 1e-5 * norm + 1e-30, err / max(norm, 1e-30)


ATTEND = [
    # lens (ctx, rows), nq, nkv, d, page
    ([(1, 1)], 32, 8, 128, 16),
    ([(2, 2)], 4, 2, 64, 16),
    ([(16, 1), (17, 1), (15, 1)], 8, 2, 128, 16),
    ([(513, 1)], 32, 8, 128, 64),
    ([(0, 0), (5, 1), (0, 0), (130, 3), (64, 0)], 8, 2, 64, 32),
    ([(1000, 1), (3, 1), (777, 1), (64, 1), (65, 1)], 28, 4, 128, 16),
    ([(300, 5), (41, 41), (256, 1)], 6, 6, 64, 256),
    ([(700, 1)], 12, 1, 128, 128),
    ([(700, 9)], 20, 1, 64, 16),
    ([(130, 130), (1, 1), (95, 33)], 8, 2, 128, 16),
    ([(257, 200), (129, 129)], 4, 4, 64, 64),
    ([(2050, 1), (31, 1)], 64, 8, 128, 64),
    ([(300, 129), (300, 128), (300, 127), (128, 128)], 2, 1, 128, 32),
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("lens,nq,nkv,d,page", ATTEND)
def test_attention(ops, lens, nq, nkv, d, page, dtype):
    rng = np.random.default_rng(len(lens) * 1000 + lens[0][0] + nq)
    table, start, ctx, total = make_batch(lens, page, rng)
    cache = random_cache(total, nkv, page, d, rng)
    poison_unused(cache, table, ctx)
    q = torch.from_numpy(rng.normal(0, 1.5, (start[-1], nq * d)).astype(np.float32)).to(dtype)
    want = ref.attention(q.double().numpy(), cache, table, start, ctx, nq, nkv, d)
    out = torch.full((start[-1], nq * d), float("nan"), dtype=dtype, device="cuda")
    got = ops.attention_kv4(q.cuda(), dev(cache), di(table), di(start), di(ctx), nq, nkv, d, out=out)
    check_attention(got, want, dtype, 4.0)
    again = ops.attention_kv4(q.cuda(), dev(cache), di(table), di(start), di(ctx), nq, nkv, d)
    assert torch.equal(got, again)  # no atomics decide a result


PROMPTS = [  # enough rows for the kernel of prompts
    ([(60, 60)], 32, 8, 128, 16),
    ([(128, 64)], 32, 8, 128, 64),
    ([(129, 65), (300, 64), (3, 1), (0, 0), (257, 63)], 32, 8, 128, 32),
    ([(200, 100), (383, 33)], 64, 8, 128, 16),
    ([(385, 129), (90, 2)], 32, 8, 64, 256),
    ([(77, 77), (400, 1), (400, 60)], 56, 8, 64, 16),
    ([(513, 100)], 16, 16, 64, 128),
    ([(130, 70)], 72, 8, 128, 16),
]


@pytest.mark.parametrize("lens,nq,nkv,d,page", PROMPTS)
def test_attention_prompts(ops, lens, nq, nkv, d, page):
    rng = np.random.default_rng(len(lens) * 100 + lens[0][0])
    table, start, ctx, total = make_batch(lens, page, rng)
    cache = random_cache(total, nkv, page, d, rng)
    poison_unused(cache, table, ctx)
    q = rng.normal(0, 1.5, (start[-1], nq * d)).astype(np.float32)
    q[0, :d] = 0
    q[-1, -d:] *= 30  # one head whose scores are far apart
    q = bf16(q)
    want = ref.attention(q.double().numpy(), cache, table, start, ctx, nq, nkv, d)
    out = torch.full((start[-1], nq * d), float("nan"), dtype=torch.bfloat16, device="cuda")
    got = ops.attention_kv4(q.cuda(), dev(cache), di(table), di(start), di(ctx), nq, nkv, d, out=out)
    check_attention(got, want, torch.bfloat16, 4.0)
    again = ops.attention_kv4(q.cuda(), dev(cache), di(table), di(start), di(ctx), nq, nkv, d)
    assert torch.equal(got, again)


MORE_PROMPTS = [  # the kernel of prompts takes over at some 400 columns (row, q head of the group) of 8 kv heads
    ([(160, 160)], 32, 8, 128, 16),
    ([(300, 128), (301, 129)], 32, 8, 64, 64),
    ([(513, 200)], 16, 16, 64, 128),
    ([(257, 130)], 32, 8, 128, 256),
    ([(128, 128), (0, 0), (2, 2)], 40, 8, 128, 32),
]


@pytest.mark.parametrize("lens,nq,nkv,d,page", MORE_PROMPTS)
def test_attention_more_prompts(ops, lens, nq, nkv, d, page):
    test_attention_prompts(ops, lens, nq, nkv, d, page)


@pytest.mark.parametrize("rows", [128, 150])
def test_attention_prompts_moving_reference(ops, rows):
    """Scores that grow along the keys, in the kernel of prompts."""
    rng = np.random.default_rng(41)
    nq, nkv, d, page = 32, 8, 128, 64
    table, start, ctx, total = make_batch([(600, rows)], page, rng)
    kc, kp, vc, vp = random_cache(total, nkv, page, d, rng)
    for i in range(600):
        kp[table[0, i // page], :, i % page, :, 1] += np.float16(0.002 * i)
    q = bf16(np.abs(rng.normal(0, 1, (rows, nq * d))))
    want = ref.attention(q.double().numpy(), (kc, kp, vc, vp), table, start, ctx, nq, nkv, d)
    got = ops.attention_kv4(q.cuda(), dev((kc, kp, vc, vp)), di(table), di(start), di(ctx), nq, nkv, d)
    got = got.double().cpu().numpy()
    # scores up to 100 from keys rounded to 11 bits: 2^-12 of them in the exponent, shared by a key's terms
    assert np.linalg.norm(got - want) <= 2.0 ** -4 * np.linalg.norm(want)


def test_attention_prompts_largest_elements(ops):
    """Elements at and beyond fp16's largest value in the kernel of prompts."""
    rng = np.random.default_rng(43)
    nq, nkv, d, page = 32, 8, 128, 16
    table, start, ctx, total = make_batch([(200, 140)], page, rng)
    kc, kp, vc, vp = random_cache(total, nkv, page, d, rng)
    vp[..., 0], vp[..., 1] = np.float16(4366), np.float16(0)
    kp[..., 0], kp[..., 1] = np.float16(4000), np.float16(-30000)
    q = bf16(rng.normal(0, 1e-5, (140, nq * d)))
    want = ref.attention(q.double().numpy(), (kc, kp, vc, vp), table, start, ctx, nq, nkv, d)
    got = ops.attention_kv4(q.cuda(), dev((kc, kp, vc, vp)), di(table), di(start), di(ctx), nq, nkv, d)
    assert np.linalg.norm(got.double().cpu().numpy() - want) <= 2.0 ** -7 * np.linalg.norm(want)
    vp[..., 1] = np.float16(30000)  # 30000 + 15 * 4366 is beyond fp16: taken as 65504
    got = ops.attention_kv4(q.cuda(), dev((kc, kp, vc, vp)), di(table), di(start), di(ctx), nq, nkv, d)
    assert torch.isfinite(got).all()


@pytest.mark.parametrize("lens", [[(32768, 1)], [(20000, 2), (9, 1)]])
def test_attention_fp32_flat_average(ops, lens):
    """An average over many keys is small beside its terms; it is held to 2e-6 of itself (p and the sums in 22 to 24
    bits, a result 2^-7 of its terms)."""
    rng = np.random.default_rng(44)
    nq, nkv, d, page = 4, 2, 64, 64
    table, start, ctx, total = make_batch(lens, page, rng)
    cache = random_cache(total, nkv, page, d, rng)
    q = torch.from_numpy(rng.normal(0, 0.3, (start[-1], nq * d)).astype(np.float32))
    want = ref.attention(q.double().numpy(), cache, table, start, ctx, nq, nkv, d)
    got = ops.attention_kv4(q.cuda(), dev(cache), di(table), di(start), di(ctx), nq, nkv, d).double().cpu().numpy()
    assert np.linalg.norm(got - want) <= 2e-6 * np.linalg.norm(want)


def test_attention_prompts_rising_scores(ops):
    """Scores that grow along the keys, so that the softmax reference moves many times."""
    rng = np.random.default_rng(31)
    nq, nkv, d, page = 32, 8, 128, 64
    table, start, ctx, total = make_batch([(700, 64)], page, rng)
    kc, kp, vc, vp = random_cache(total, nkv, page, d, rng)
    for i in range(700):
        kp[table[0, i // page], :, i % page, :, 1] += np.float16(0.01 * i)
    q = bf16(np.abs(rng.normal(0, 1, (64, nq * d))))
    want = ref.attention(q.double().numpy(), (kc, kp, vc, vp), table, start, ctx, nq, nkv, d)
    got = ops.attention_kv4(q.cuda(), dev((kc, kp, vc, vp)), di(table), di(start), di(ctx), nq, nkv, d)
    got = got.double().cpu().numpy()
    # scores of hundreds from keys rounded to 11 bits: an absolute error of some 2^-5 in the exponent
    assert np.linalg.norm(got - want) <= 2.0 ** -4 * np.linalg.norm(want)


def test_attention_prompts_strides_and_missing_pages(ops):
    """Unaligned rows, a page that is none and a context past the page table, with many rows."""
    rng = np.random.default_rng(32)
    nq, nkv, d, page = 32, 8, 64, 16
    table, start, ctx, total = make_batch([(300, 70), (20, 40)], page, rng, pages=19)
    cache = random_cache(total, nkv, page, d, rng)
    table[0, 2], table[0, 9] = -3, total + 5
    ctx[0] = 19 * 16 + 9
    wide = bf16(rng.normal(0, 1, (110, nq * d + 7))).cuda()
    q = wide[:, 3: 3 + nq * d]
    want = ref.attention(q.double().cpu().numpy(), cache, table, start, ctx, nq, nkv, d)
    out = torch.zeros(110, nq * d + 5, dtype=torch.bfloat16, device="cuda")
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    ops.attention_kv4(q, dev(cache), di(table), di(start), di(ctx), nq, nkv, d, out=out[:, 1: 1 + nq * d],
                      status=status)
    check_attention(out[:, 1: 1 + nq * d], want, torch.bfloat16, 4.0)
    assert (out[:, 0] == 0).all() and (out[:, 1 + nq * d:] == 0).all()
    assert (out[start[1]: start[1] + 20] == 0).all()
    assert status.item() == 11


def test_attention_prompts_largest_values(ops):
    """Elements at and beyond fp16's largest value stay finite."""
    rng = np.random.default_rng(33)
    nq, nkv, d, page = 32, 8, 128, 16
    table, start, ctx, total = make_batch([(100, 60)], page, rng)
    kc, kp, vc, vp = random_cache(total, nkv, page, d, rng)
    vp[..., 0], vp[..., 1] = np.float16(4366), np.float16(0)
    kp[..., 0], kp[..., 1] = np.float16(4000), np.float16(-30000)
    q = bf16(rng.normal(0, 1e-5, (60, nq * d)))
    want = ref.attention(q.double().numpy(), (kc, kp, vc, vp), table, start, ctx, nq, nkv, d)
    got = ops.attention_kv4(q.cuda(), dev((kc, kp, vc, vp)), di(table), di(start), di(ctx), nq, nkv, d)
    assert np.linalg.norm(got.double().cpu().numpy() - want) <= 2.0 ** -7 * np.linalg.norm(want)
    vp[..., 1] = np.float16(30000)  # 30000 + 15 * 4366 is beyond fp16: taken as 65504
    got = ops.attention_kv4(q.cuda(), dev((kc, kp, vc, vp)), di(table), di(start), di(ctx), nq, nkv, d)
    assert torch.isfinite(got).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("big", [1.0, 60.0])
def test_attention_sharp_and_flat(ops, dtype, big):
    """Scores that differ by hundreds (one key takes all) and a zero q (every key alike)."""
    rng = np.random.default_rng(5)
    table, start, ctx, total = make_batch([(333, 2), (90, 1)], 16, rng)
    cache = random_cache(total, 2, 16, 128, rng)
    q = rng.normal(0, big, (3, 8 * 128)).astype(np.float32)
    q[1] = 0
    q[2, :128] *= 1e-3
    q = torch.from_numpy(q).to(dtype)
    want = ref.attention(q.double().numpy(), cache, table, start, ctx, 8, 2, 128)
    got = ops.attention_kv4(q.cuda(), dev(cache), di(table), di(start), di(ctx), 8, 2, 128)
    got = got.double().cpu().numpy()
    # scores of hundreds: an absolute error of 2^-14 of them in p
    tol = {torch.bfloat16: 2.0 ** -7, torch.float32: 1e-5 * max(1.0, big)}[dtype]
    assert np.linalg.norm(got - want) <= tol * np.linalg.norm(want)


def test_attention_extreme_scales(ops):
    """Values from the smallest fp16 scales to the largest, q from 1e-6 to 1e4."""
    rng = np.random.default_rng(8)
    for s, m, qs in ((6e-8, 0.0, 1e4), (1e-4, 1e-3, 100.0), (1000.0, -7500.0, 1e-5), (4300.0, 0.0, 1e-6)):
        table, start, ctx, total = make_batch([(150, 1)], 16, rng)
        kc, kp, vc, vp = random_cache(total, 1, 16, 128, rng)
        for p in (kp, vp):
            p[..., 0], p[..., 1] = np.float16(s), np.float16(m)
        q = bf16(rng.normal(0, qs, (1, 4 * 128)))
        want = ref.attention(q.double().numpy(), (kc, kp, vc, vp), table, start, ctx, 4, 1, 128)
        got = ops.attention_kv4(q.cuda(), dev((kc, kp, vc, vp)), di(table), di(start), di(ctx), 4, 1, 128)
        got = got.double().cpu().numpy()
        assert np.isfinite(got).all()
        assert np.linalg.norm(got - want) <= 2.0 ** -7 * np.linalg.norm(want) + 1e-7 * 15 * s


@pytest.mark.parametrize("rows", [1, 40])
def test_attention_missing_pages_and_lengths(ops, rows):
    """Pages outside the cache are masked and reported; a context below its rows leaves rows that see nothing."""
    rng = np.random.default_rng(9)
    lens = [(200, rows), (rows // 2, rows), (100, rows)]
    table, start, ctx, total = make_batch(lens, 16, rng, pages=14)
    cache = random_cache(total, 2, 16, 64, rng)
    table[0, 3], table[0, 7] = -1, total
    ctx[2] = 14 * 16 + 50  # past the page table: keys there do not exist
    table[2, :14] = table[0, :14]
    q = bf16(rng.normal(0, 1, (start[-1], 8 * 64)))
    want = ref.attention(q.double().numpy(), cache, table, start, ctx, 8, 2, 64)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    got = ops.attention_kv4(q.cuda(), dev(cache), di(table), di(start), di(ctx), 8, 2, 64, status=status)
    check_attention(got, want, torch.bfloat16, 4.0)
    assert status.item() == 11  # OUT_OF_RANGE
    if rows // 2 < rows:
        assert (got[start[1]: start[1] + rows - rows // 2] == 0).all()


def test_attention_strides_scale_and_stream(ops):
    """q a slice of a wider row, out strided, planes of one allocation, another stream, another scale."""
    rng = np.random.default_rng(10)
    nq, nkv, d, page = 8, 2, 128, 32
    table, start, ctx, total = make_batch([(210, 1), (70, 3)], page, rng)
    cache = random_cache(total, nkv, page, d, rng)
    both_c = torch.zeros(total, 2, nkv, page, d // 2, dtype=torch.uint8, device="cuda")
    both_p = torch.zeros(total, 2, nkv, page, d // 64, 2, dtype=torch.float16, device="cuda")
    for i in (0, 1):
        both_c[:, i] = torch.from_numpy(cache[2 * i]).cuda()
        both_p[:, i] = torch.from_numpy(cache[2 * i + 1]).cuda()
    wide = bf16(rng.normal(0, 1, (4, nq * d + 2 * nkv * d + 6))).cuda()
    q = wide[:, 6: 6 + nq * d]
    out = torch.zeros(4, nq * d + 3, dtype=torch.bfloat16, device="cuda")[:, 1: 1 + nq * d]
    want = ref.attention(q.double().cpu().numpy(), cache, table, start, ctx, nq, nkv, d, scale=0.03)
    args = (di(table), di(start), di(ctx))
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        ops.attention_kv4(q, (both_c[:, 0], both_p[:, 0], both_c[:, 1], both_p[:, 1]), *args, nq, nkv, d, scale=0.03,
                          out=out)
    s.synchronize()
    check_attention(out, want, torch.bfloat16, 4.0)


def test_attention_long_cache_offsets(ops):
    """Pages beyond 2^32 bytes of a plane."""
    rng = np.random.default_rng(11)
    nkv, d, page = 8, 128, 256
    per = nkv * page * d // 2
    total = (1 << 32) // per + 40
    kc = torch.zeros(total, nkv, page, d // 2, dtype=torch.uint8, device="cuda")
    kp = torch.zeros(total, nkv, page, 2, 2, dtype=torch.float16, device="cuda")
    small = random_cache(4, nkv, page, d, rng)
    at = np.array([total - 1, total - 30, 1, total - 3])
    kc[at], kp[at] = torch.from_numpy(small[0]).cuda(), torch.from_numpy(small[1]).cuda()
    vp = kp.clone()
    table = at.astype(np.int32)[None]
    start, ctx = np.array([0, 1], np.int32), np.array([1000], np.int32)
    q = bf16(rng.normal(0, 1, (1, 8 * d)))
    want = ref.attention(q.double().numpy(), (small[0], small[1], small[0], small[1]),
                         np.arange(4, dtype=np.int32)[None], start, ctx, 8, nkv, d)
    got = ops.attention_kv4(q.cuda(), (kc, kp, kc, vp), di(table), di(start), di(ctx), 8, nkv, d)
    check_attention(got, want, torch.bfloat16, 4.0)


def test_attention_many_sequences(ops):
    """More sequences than threads in a block, most of one token, some empty."""
    rng = np.random.default_rng(12)
    lens = [(int(c), 1 if c else 0) for c in rng.integers(0, 40, 700)]
    lens[650] = (900, 4)
    table, start, ctx, total = make_batch(lens, 16, rng)
    cache = random_cache(total, 1, 16, 64, rng)
    q = bf16(rng.normal(0, 1, (start[-1], 4 * 64)))
    want = ref.attention(q.double().numpy(), cache, table, start, ctx, 4, 1, 64)
    got = ops.attention_kv4(q.cuda(), dev(cache), di(table), di(start), di(ctx), 4, 1, 64)
    check_attention(got, want, torch.bfloat16, 4.0)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("n,longest,nq,nkv,d,page", [
    (120, 380, 32, 8, 128, 16),   # each warp takes whole items
    (120, 384, 32, 8, 128, 64),
    (120, 2000, 32, 8, 128, 64),  # a long one among them: shares of all units
    (700, 60, 12, 1, 64, 32),
    (90, 33, 20, 10, 64, 16),
])
def test_attention_many_short_sequences(ops, n, longest, nq, nkv, d, page, dtype):
    rng = np.random.default_rng(n + longest + d)
    lens = [(int(c), int(min(c, r))) for c, r in zip(rng.integers(0, min(longest, 380) + 1, n), rng.integers(0, 4, n))]
    lens[n // 3] = (longest, 1)
    lens[-1] = (longest, 2)
    lens[0] = (1, 1)
    table, start, ctx, total = make_batch(lens, page, rng)
    cache = random_cache(total, nkv, page, d, rng)
    poison_unused(cache, table, ctx)
    q = torch.from_numpy(rng.normal(0, 1.5, (start[-1], nq * d)).astype(np.float32)).to(dtype)
    want = ref.attention(q.double().numpy(), cache, table, start, ctx, nq, nkv, d)
    out = torch.full((start[-1], nq * d), float("nan"), dtype=dtype, device="cuda")
    got = ops.attention_kv4(q.cuda(), dev(cache), di(table), di(start), di(ctx), nq, nkv, d, out=out)
    check_attention(got, want, dtype, 4.0)
    assert torch.equal(got, ops.attention_kv4(q.cuda(), dev(cache), di(table), di(start), di(ctx), nq, nkv, d))


def test_attention_many_short_sequences_missing_pages(ops):
    rng = np.random.default_rng(19)
    lens = [(int(c), 1) for c in rng.integers(1, 129, 150)]
    lens[7] = (2, 5)  # a context below its rows
    table, start, ctx, total = make_batch(lens, 16, rng, pages=8)
    cache = random_cache(total, 8, 16, 64, rng)
    table[3, 0], table[20, :] = -1, total + 5  # the first page of one, all of another
    ctx[50] = 8 * 16 + 9  # past the page table
    table[50] = table[51]
    q = bf16(rng.normal(0, 1, (start[-1], 32 * 64)))
    want = ref.attention(q.double().numpy(), cache, table, start, ctx, 32, 8, 64)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    got = ops.attention_kv4(q.cuda(), dev(cache), di(table), di(start), di(ctx), 32, 8, 64, status=status)
    check_attention(got, want, torch.bfloat16, 4.0)
    assert status.item() == 11  # OUT_OF_RANGE
    assert (got[start[20]] == 0).all() and (got[start[7]: start[7] + 3] == 0).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("ctx,rows", [(1, 1), (7, 2), (20, 1), (120, 3)])
@pytest.mark.parametrize("nq,nkv,d", [(32, 8, 128), (56, 8, 64), (16, 16, 64)])
def test_attention_few_keys(ops, ctx, rows, nq, nkv, d, dtype):
    """Items of fewer units than a CTA has warps."""
    rng = np.random.default_rng(ctx * 10 + rows + nq)
    table, start, lens, total = make_batch([(ctx, rows)], 16, rng)
    cache = random_cache(total, nkv, 16, d, rng)
    poison_unused(cache, table, lens)
    q = torch.from_numpy(rng.normal(0, 1.5, (rows, nq * d)).astype(np.float32)).to(dtype)
    want = ref.attention(q.double().numpy(), cache, table, start, lens, nq, nkv, d)
    got = ops.attention_kv4(q.cuda(), dev(cache), di(table), di(start), di(lens), nq, nkv, d)
    check_attention(got, want, dtype, 4.0)


# ------------------------------------------------------------------ append and gather
APPEND = [
    # lens (ctx, rows), nq, nkv, d, page
    ([(1, 1)], 32, 8, 128, 16),
    ([(513, 1), (16, 1), (17, 1)], 4, 2, 64, 16),
    ([(40, 40), (0, 0), (33, 5), (7, 1)], 8, 2, 128, 32),
    ([(300, 130)], 3, 1, 64, 256),
    ([(129, 64)], 5, 5, 128, 128),
]


def append_inputs(lens, nq, nkv, d, page, dtype, seed):
    rng = np.random.default_rng(seed)
    table, start, ctx, total = make_batch(lens, page, rng)
    rows = start[-1]
    x = rng.normal(0, 1, (rows, (nq + 2 * nkv) * d)).astype(np.float32)
    x[:, ::41] *= 5
    x = torch.from_numpy(x).to(dtype).cuda()
    q, k, v = x[:, : nq * d], x[:, nq * d: (nq + nkv) * d], x[:, (nq + nkv) * d:]
    cs = ref.rope_table(10000.0, d, max(1, max(ctx)))
    b = np.repeat(np.arange(len(lens)), np.diff(start))
    pos = ctx[b] - start[b + 1] + np.arange(rows)
    return rng, table, start, ctx, total, q, k, v, cs, b, pos


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("lens,nq,nkv,d,page", APPEND)
def test_append_bit_exact_without_norm(ops, lens, nq, nkv, d, page, dtype):
    rng, table, start, ctx, total, q, k, v, cs, b, pos = append_inputs(lens, nq, nkv, d, page, dtype, 21)
    cache = ops.kv4_cache(total, page, nkv, d)
    for c in cache:
        c.view(torch.uint8).fill_(0xA5)
    before = [c.cpu().numpy().copy() for c in cache]
    out = ops.kv4_append(q, k, v, cache, di(table), di(start), di(ctx), torch.from_numpy(cs).cuda(), nq, nkv, d)
    at, slot = table[b, pos // page], pos % page
    rot = {}
    for name, t, n in (("q", q, nq), ("k", k, nkv)):
        rot[name] = ref.norm_rotate(t.float().cpu().numpy().reshape(len(pos), n, d), None, cs[pos], 0)
    vals = v.float().cpu().numpy().reshape(len(pos), nkv, d)
    torch.testing.assert_close(out.cpu(), torch.from_numpy(rot["q"].reshape(len(pos), -1)).to(dtype), rtol=0, atol=0)
    for i, x in ((0, rot["k"]), (2, vals)):
        code, par = ref.quantise(x)
        want_c, want_p = before[i], before[i + 1]
        want_c[at, :, slot], want_p[at, :, slot] = ref.pack_rows(code), par
        np.testing.assert_array_equal(cache[i].cpu().numpy(), want_c)
        np.testing.assert_array_equal(cache[i + 1].cpu().numpy().view(np.uint16), want_p.view(np.uint16))
    # read back
    for out_t in (torch.bfloat16, torch.float32):
        gk, gv = ops.kv4_gather(cache, di(table), di(start), di(ctx), len(pos), nkv, d, dtype=out_t)
        for got, x in ((gk, rot["k"]), (gv, vals)):
            code, par = ref.quantise(x)
            want = torch.from_numpy(ref.values(ref.pack_rows(code), par).reshape(len(pos), -1))
            torch.testing.assert_close(got.cpu(), want.float().to(out_t), rtol=0 if out_t != torch.float32 else 1e-7,
                                       atol=0 if out_t != torch.float32 else 1e-7)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("lens,nq,nkv,d,page", APPEND)
def test_append_with_norms(ops, lens, nq, nkv, d, page, dtype):
    rng, table, start, ctx, total, q, k, v, cs, b, pos = append_inputs(lens, nq, nkv, d, page, dtype, 22)
    qw, kw = (torch.from_numpy(rng.normal(1, 0.2, d).astype(np.float32)).to(dtype).cuda() for _ in range(2))
    cache = ops.kv4_cache(total, page, nkv, d)
    qc = q.clone()
    out = ops.kv4_append(qc, k, v, cache, di(table), di(start), di(ctx), torch.from_numpy(cs).cuda(), nq, nkv, d,
                         q_norm=qw, k_norm=kw, eps=1e-6, q_out=qc)
    assert out.data_ptr() == qc.data_ptr()
    want = ref.norm_rotate(q.double().cpu().numpy().reshape(len(pos), nq, d), qw.double().cpu().numpy(),
                           cs[pos].astype(np.float64), 1e-6).reshape(len(pos), -1)
    # fp32: the norm's factor and two products to a few 2^-24 each, then a difference of them
    tol = 2.0 ** -8 if dtype == torch.bfloat16 else 2e-6
    np.testing.assert_allclose(out.double().cpu().numpy(), want, rtol=tol, atol=1e-6 * np.abs(want).max())
    x = ref.norm_rotate(k.double().cpu().numpy().reshape(len(pos), nkv, d), kw.double().cpu().numpy(),
                        cs[pos].astype(np.float64), 1e-6)
    code, par = ref.quantise(x)
    at, slot = table[b, pos // page], pos % page
    got_p = cache[1].cpu().numpy()[at, :, slot]
    assert (np.abs(got_p.astype(np.float64) - par) <= np.spacing(np.abs(par)).astype(np.float64)).all()
    got_c = ref.unpack_rows(cache[0].cpu().numpy()[at, :, slot]).astype(int)
    # the quotient with the parameters that were written: a code is off only next to a half
    s, m = (np.repeat(got_p[..., j].astype(np.float64), 64, -1) for j in (0, 1))
    quot = (x - m) / s
    assert (np.abs(got_c - np.clip(quot, 0, 15)) <= 0.5 + 2.0 ** -8).all()


def test_append_edge_values(ops):
    """Constant groups, zeros, values beyond fp16, NaN and infinity stay where they are."""
    d, nq, nkv, page = 64, 1, 1, 16
    rows = 6
    x = np.random.default_rng(3).normal(0, 1, (rows, d)).astype(np.float32)
    x[0] = 0.0
    x[1] = 3.25
    x[2, 5] = 1e30
    x[3, 7] = -1e30
    x[4, 9] = np.nan
    x[5, 0], x[5, 1] = np.inf, -np.inf
    cs = np.zeros((rows, d // 2, 2), np.float32)
    cs[..., 0] = 1  # no rotation
    cache = ops.kv4_cache(2, page, nkv, d)
    xt = torch.from_numpy(x).cuda()
    args = [torch.tensor(a, dtype=torch.int32, device="cuda") for a in ([[1]], [0, rows], [rows])]
    ops.kv4_append(xt, xt, xt, cache, *args, torch.from_numpy(cs).cuda(), nq, nkv, d)
    k, v = (t.cpu().numpy() for t in ops.kv4_gather(cache, *args, rows, nkv, d, dtype=torch.float32))
    np.testing.assert_array_equal(v[0], 0)
    np.testing.assert_array_equal(v[1], 3.25)
    assert np.isfinite(v).all()
    assert v[2].argmax() == 5 and abs(v[2, 5] - (15 * 4366 + v[2].min())) < 32
    assert v[3, 7] == -65504
    fine = np.delete(np.arange(d), 9)
    lo, hi = x[4, fine].min(), x[4, fine].max()
    assert np.abs(v[4, fine] - x[4, fine]).max() <= (hi - lo) / 30 * 1.01 + 1e-3
    assert v[4, 9] == v[4].min()
    assert v[5, 0] == v[5].max() and v[5, 1] == -65504
    np.testing.assert_array_equal(k[:2], v[:2])
    np.testing.assert_array_equal((cache[0][0] != 0).sum().item(), 0)  # page 0 untouched


def test_append_out_of_range_rows(ops):
    """Rows before position 0, past the table, past the rotation table or on a page that is none write nothing."""
    rng = np.random.default_rng(4)
    d, nq, nkv, page = 64, 2, 1, 16
    table = np.array([[0, 9], [1, 2], [3, 4]], np.int32)  # 9 is no page
    start, ctx = np.array([0, 4, 8, 12], np.int32), np.array([18, 2, 34], np.int32)
    x = torch.from_numpy(rng.normal(0, 1, (12, 4 * d)).astype(np.float32)).cuda()
    cs = torch.from_numpy(ref.rope_table(10000.0, d, 33)).cuda()
    cache = ops.kv4_cache(5, page, nkv, d)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    ops.kv4_append(x[:, : 2 * d], x[:, 2 * d: 3 * d], x[:, 3 * d:], cache, di(table), di(start), di(ctx), cs, nq, nkv,
                   d, status=status)
    assert status.item() == 11
    written = (cache[1].float().abs().sum((1, 3, 4)) > 0).cpu().numpy()
    want = np.zeros((5, page), bool)
    want[0, 14:16] = True    # sequence 0: positions 14, 15 (16, 17 have no page)
    want[1, 0:2] = True      # sequence 1: positions -2, -1 are none
    want[4, 14:16] = True    # sequence 2: positions 30, 31 (32, 33: past the page table)
    np.testing.assert_array_equal(written, want)
    status.zero_()
    k, _ = ops.kv4_gather(cache, di(table), di(start), di(ctx), 12, nkv, d, status=status)
    assert status.item() == 11
    zero = (k == 0).all(1).cpu().numpy()
    np.testing.assert_array_equal(zero, [False, False, True, True, True, True, False, False, False, False, True, True])


def test_append_then_attend_one_token_at_a_time(ops):
    """A conversation built token by token reads like one appended at once."""
    rng = np.random.default_rng(6)
    nq, nkv, d, page, n = 8, 2, 128, 16, 37
    x = bf16(rng.normal(0, 1, (n, (nq + 2 * nkv) * d))).cuda()
    q, k, v = x[:, : nq * d], x[:, nq * d: (nq + nkv) * d], x[:, (nq + nkv) * d:]
    cs = torch.from_numpy(ref.rope_table(500000.0, d, n)).cuda()
    table = torch.tensor([[2, 0, 3]], dtype=torch.int32, device="cuda")

    def call(cache, lo, hi):
        st = torch.tensor([0, hi - lo], dtype=torch.int32, device="cuda")
        cl = torch.tensor([hi], dtype=torch.int32, device="cuda")
        qr = ops.kv4_append(q[lo:hi], k[lo:hi], v[lo:hi], cache, table, st, cl, cs, nq, nkv, d)
        return ops.attention_kv4(qr, cache, table, st, cl, nq, nkv, d)

    one, many = ops.kv4_cache(4, page, nkv, d), ops.kv4_cache(4, page, nkv, d)
    whole = call(one, 0, n)
    parts = torch.cat([call(many, i, i + 1) for i in range(n)])
    for a, b in zip(one, many):
        assert torch.equal(a, b)
    err = (whole.double() - parts.double()).norm() / whole.double().norm()
    assert err <= 2.0 ** -7  # two roundings to bf16


def test_empty_calls(ops):
    cache = ops.kv4_cache(1, 16, 1, 64)
    none = torch.zeros(0, 64, dtype=torch.bfloat16, device="cuda")
    for n_seq in (0, 2):
        table = torch.zeros(n_seq, 1, dtype=torch.int32, device="cuda")
        start = torch.zeros(n_seq + 1, dtype=torch.int32, device="cuda")
        ctx = torch.zeros(n_seq, dtype=torch.int32, device="cuda")
        cs = torch.zeros(1, 32, 2, device="cuda")
        assert ops.kv4_append(none, none, none, cache, table, start, ctx, cs, 1, 1, 64).shape == (0, 64)
        assert ops.attention_kv4(none, cache, table, start, ctx, 1, 1, 64).shape == (0, 64)
        assert ops.kv4_gather(cache, table, start, ctx, 0, 1, 64)[0].shape == (0, 64)


def test_front_end_refusals(ops):
    cache = ops.kv4_cache(2, 16, 2, 64)
    q = torch.zeros(1, 4 * 64, dtype=torch.bfloat16, device="cuda")
    ints = [torch.tensor(a, dtype=torch.int32, device="cuda") for a in ([[0]], [0, 1], [1])]
    with pytest.raises(ValueError):
        ops.attention_kv4(q.cpu(), cache, *ints, 4, 2, 64)
    with pytest.raises(ValueError):
        ops.attention_kv4(q, cache, *ints, 4, 1, 64)       # the cache has two heads
    with pytest.raises(ValueError):
        ops.attention_kv4(q[:, :64], cache, *ints, 4, 2, 64)
    with pytest.raises(ValueError):
        ops.attention_kv4(q, cache, ints[0].long(), *ints[1:], 4, 2, 64)
    with pytest.raises(ValueError):
        ops.attention_kv4(q, cache, ints[0], ints[1][:1], ints[2], 4, 2, 64)
    with pytest.raises(ValueError):
        ops.kv4_append(q, q, q, cache, *ints, torch.zeros(1, 32, 2, device="cuda"), 4, 2, 64)
    from aethermind_b200 import AmError
    with pytest.raises(AmError):
        ops.attention_kv4(q[:, :192], cache, *ints, 3, 2, 64)  # 3 query heads over 2
