"""The 4-bit cache's and the sampler's checks of arguments, on the host (no GPU)."""
import ctypes as C

import numpy as np
import pytest

import kv4_reference as ref


def attention_args(L, **change):
    a = L.AmcuKv4AttentionArgs()
    a.cache = L.AmcuKv4Cache(4096, 4096, 4096, 4096, 0, 0, 8, 16, 2, 128)
    a.batch = L.AmcuKv4Batch(4096, 0, 4, 4096, 4096, 1, 1, None)
    a.q = a.out = 4096
    a.q_stride = a.out_stride = 4 * 128
    a.n_q_heads, a.dtype = 4, L.BF16
    for k, v in change.items():
        o, *rest = k.split("__")
        setattr(getattr(a, o), rest[0], v) if rest else setattr(a, o, v)
    return a


@pytest.mark.parametrize("change,word", [
    (dict(cache__head_dim=96), b"head_dim"), (dict(cache__head_dim=0), b"head_dim"),
    (dict(cache__page_size=8), b"page_size"), (dict(cache__page_size=48), b"page_size"),
    (dict(cache__page_size=512), b"page_size"), (dict(cache__n_kv_heads=0), b"n_kv_heads"),
    (dict(cache__num_pages=0), b"num_pages"), (dict(cache__num_pages=1 << 31), b"num_pages"),
    (dict(cache__k_codes=None), b"null"), (dict(cache__v_params=4104), b"aligned"),
    (dict(cache__codes_page_stride=2040), b"codes_page_stride"),
    (dict(cache__codes_page_stride=2056), b"codes_page_stride"),
    (dict(cache__params_page_stride=16), b"params_page_stride"),
    (dict(batch__rows=-1), b"rows"), (dict(batch__n_seq=-1), b"n_seq"), (dict(batch__rows=1 << 25), b"rows"),
    (dict(batch__row_start=None), b"null"), (dict(batch__ctx_len=None), b"null"),
    (dict(batch__page_table=None), b"null"), (dict(batch__max_pages=-1), b"max_pages"),
    (dict(batch__n_seq=2, batch__table_stride=3), b"table_stride"),
    (dict(n_q_heads=3), b"n_q_heads"), (dict(n_q_heads=0), b"n_q_heads"), (dict(dtype=2), b"dtype"),
    (dict(q=None), b"null"), (dict(out=None), b"null"), (dict(scale=float("nan")), b"scale"),
    (dict(scale=-1.0), b"scale"), (dict(scale=float("inf")), b"scale"),
])
def test_attention_refusals(built_lib, change, word):
    from aethermind_b200 import _lib as L
    assert built_lib.amcu_attn_kv4(C.byref(attention_args(L, **change)), None) == 3
    msg = built_lib.amcu_last_error()
    assert b"amcu_attn_kv4" in msg and word in msg


@pytest.mark.parametrize("change,word", [
    (dict(dtype=2), b"dtype"), (dict(n_q_heads=0), b"n_q_heads"), (dict(max_pos=0), b"max_pos"),
    (dict(eps=-1.0), b"eps"), (dict(eps=float("nan")), b"eps"), (dict(k=None), b"null"), (dict(cos_sin=None), b"null"),
    (dict(q=4098), b"two-element"), (dict(v_stride=257), b"two-element"), (dict(k_norm=4097), b"two-element"),
    (dict(cos_sin=4104), b"cos_sin"), (dict(cache__page_size=24), b"page_size"),
])
def test_append_refusals(built_lib, change, word):
    from aethermind_b200 import _lib as L
    a = L.AmcuKv4AppendArgs()
    base = attention_args(L)
    a.cache, a.batch = base.cache, base.batch
    a.q = a.k = a.v = a.q_out = a.cos_sin = 4096
    a.q_stride = a.q_out_stride = 512
    a.k_stride = a.v_stride = 256
    a.eps, a.dtype, a.max_pos, a.n_q_heads = 1e-5, L.BF16, 64, 4
    for k, v in change.items():
        o, *rest = k.split("__")
        setattr(getattr(a, o), rest[0], v) if rest else setattr(a, o, v)
    assert built_lib.amcu_kv4_append(C.byref(a), None) == 3
    msg = built_lib.amcu_last_error()
    assert b"amcu_kv4_append" in msg and word in msg


def test_gather_and_empty_calls(built_lib):
    from aethermind_b200 import _lib as L
    g = L.AmcuKv4GatherArgs()
    base = attention_args(L)
    g.cache, g.batch, g.dtype = base.cache, base.batch, L.BF16
    assert built_lib.amcu_kv4_gather(C.byref(g), None) == 3  # no outputs
    g.k_out = g.v_out = 4096
    g.k_out_stride = g.v_out_stride = 252
    assert built_lib.amcu_kv4_gather(C.byref(g), None) == 3
    assert b"16-byte" in built_lib.amcu_last_error()
    for change in (dict(batch__rows=0), dict(batch__n_seq=0)):  # nothing to do, nothing touched
        assert built_lib.amcu_attn_kv4(C.byref(attention_args(L, **change)), None) == 0
    for f in ("amcu_attn_kv4", "amcu_kv4_append", "amcu_kv4_gather", "amcu_sample"):
        assert getattr(built_lib, f)(None, None) == 3


@pytest.mark.parametrize("change,word", [
    (dict(rows=-1), b"rows"), (dict(vocab=0), b"vocab"), (dict(vocab=(1 << 22) + 1), b"vocab"),
    (dict(row_stride=99), b"row_stride"), (dict(dtype=2), b"dtype"), (dict(logits=None), b"null"),
    (dict(uniform=None), b"null"), (dict(out_index=None), b"null"),
])
def test_sample_refusals(built_lib, change, word):
    from aethermind_b200 import _lib as L
    a = L.AmcuSampleArgs(4096, 0, 2, 100, L.BF16, 4096, None, None, None, None, 4096, None)
    for k, v in change.items():
        setattr(a, k, v)
    assert built_lib.amcu_sample(C.byref(a), None) == 3
    assert word in built_lib.amcu_last_error()
    a = L.AmcuSampleArgs(None, 0, 0, 100, L.BF16, None, None, None, None, None, None, None)
    assert built_lib.amcu_sample(C.byref(a), None) == 0


def test_reference_rows_round_trip():
    rng = np.random.default_rng(0)
    for d in (64, 128):
        c = rng.integers(0, 16, (5, d)).astype(np.uint8)
        b = ref.pack_rows(c)
        np.testing.assert_array_equal(ref.unpack_rows(b), c)
        # element 0 is in the first byte's low nibble; with two groups the second word is the second group's
        assert (b[:, 0] & 15 == c[:, 0]).all() and (b[:, 0] >> 4 == c[:, 1]).all()
        assert (b[:, 4] & 15 == c[:, 64 if d == 128 else 8]).all()
    x = rng.normal(0, 1, (9, 128)).astype(np.float32)
    code, par = ref.quantise(x)
    v = ref.values(ref.pack_rows(code), par)
    span = x.reshape(9, 2, 64).max(-1) - x.reshape(9, 2, 64).min(-1)
    assert (np.abs(v - x).reshape(9, 2, 64).max(-1) <= span / 30 * 1.01 + 2e-3).all()


def test_front_end_wants_cuda_tensors(built_lib):
    torch = pytest.importorskip("torch")
    from aethermind_b200 import ops
    x, i = torch.zeros(2, 64), torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError):
        ops.sample(x, x[0])
    with pytest.raises(ValueError):
        ops.attention_kv4(x, (i, i, i, i), i, i, i, 1, 1, 64)
    with pytest.raises(ValueError):
        ops.kv4_append(None, x, x, (i, i, i, i), i, i, i, x, 1, 1, 64)
    with pytest.raises(ValueError):
        ops.kv4_gather((i, i, i, i), i, i, i, 2, 1, 64)
    with pytest.raises(ValueError):
        ops.kv4_gather((i, i, i, i), i, i, i, 2, 1, 64, dtype=torch.float64)
