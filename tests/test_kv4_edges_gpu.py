"""The 4-bit paged KV cache where calls go wrong: positions that do not exist, numbers that are none, rows of which one
token has nearly all the mass, and calls large enough for the kernels of prompts."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

import kv4_reference as ref  # noqa: E402
from test_kv4_gpu import bf16, dev, di, make_batch, random_cache  # noqa: E402

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
