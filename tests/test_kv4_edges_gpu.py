"""The 4-bit paged KV cache where calls go wrong: positions that do not exist, numbers that are none, rows of which one
token has nearly all the mass, and calls large enough for the kernels of prompts."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

import kv4_reference as ref  # noqa: E402
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
