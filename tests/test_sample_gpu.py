"""amcu_sample against a plain 64-bit implementation of its definition.

The weights are whole numbers of 2^-40 from a 32-bit exp (relative error below 2^-21 with the rounding of z), so a
64-bit reference names the same token wherever the draw is further than that from a border between two tokens: the
uniform numbers and the top-p limits of these tests sit in the middle of a token's share. Probabilities: 2e-5, for
|z| up to 100 rounded to 24 bits.
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


def draw_case(x, rng, t, k, min_p, nucleus):
    """top_p and a uniform number that sit clear of every border, and the token and probability they stand for."""
    top_p = 1.0
    if nucleus:
        kept, order = ref.sample_kept(x, t, k, 1.0, min_p)
        ws = kept[order]
        ws = ws[ws > 0]
        n = int(rng.integers(1, len(ws) + 1))
        while n < len(ws) and ws[n - 1] / ws.sum() < 2e-6:
            n += 1
        n = n if ws[n - 1] / ws.sum() >= 2e-6 else 1
        cum = np.cumsum(ws) / ws.sum()
        top_p = float(np.float32((cum[n - 1] + (cum[n - 2] if n > 1 else 0)) / 2))
    kept, order = ref.sample_kept(x, t, k, top_p, min_p)
    share = kept / kept.sum()
    likely = np.flatnonzero(share > 4e-6)
    token = int(rng.choice(likely))
    u = float(np.float32(share[:token].sum() + share[token] / 2))
    return top_p, u, token, share[token]


def run(ops, x, t, k, p, m, u, dtype=torch.float32, with_prob=True):
    f = lambda a: torch.tensor(a, dtype=torch.float32, device="cuda")  # noqa: E731
    x = x if torch.is_tensor(x) else torch.from_numpy(x).to(dtype).cuda()
    return ops.sample(x, f(u), temperature=f(t), top_k=torch.tensor(k, dtype=torch.int32, device="cuda"), top_p=f(p),
                      min_p=f(m), with_prob=with_prob)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("vocab,rows", [(1, 3), (2, 5), (31, 40), (509, 33), (4097, 12), (32000, 9), (128256, 6),
                                        (128255, 3), (300001, 2)])
def test_tokens_and_probabilities(ops, vocab, rows, dtype):
    rng = np.random.default_rng(vocab + rows)
    x = torch.from_numpy(rng.normal(0, 2.5, (rows, vocab)).astype(np.float32)).to(dtype).float().numpy()
    t, k, p, m, u, want, prob = [], [], [], [], [], [], []
    for i in range(rows):
        t.append(float(np.float32(rng.choice([0.0, 0.25, 0.7, 1.0, 3.0]))))
        k.append(int(rng.choice([0, 1, 2, 40, vocab, vocab + 5, max(1, vocab // 3)])))
        # a min-p of half a step between weights far apart: well away from any weight
        m.append(float(np.float32(rng.choice([0.0, 0.0, 0.031]))))
        pi, ui, tok, pr = draw_case(x[i], rng, t[-1], k[-1], m[-1], rng.random() < 0.6)
        p.append(pi), u.append(ui), want.append(tok), prob.append(pr)
    got, gp = run(ops, x, t, k, p, m, u, dtype)
    assert got.tolist() == want
    np.testing.assert_allclose(gp.cpu().numpy(), prob, rtol=2e-5)
    again, _ = run(ops, x, t, k, p, m, u, dtype)
    assert torch.equal(got, again)


def test_greedy_is_argmax(ops):
    rng = np.random.default_rng(1)
    x = torch.from_numpy(rng.normal(0, 1, (20, 5003)).astype(np.float32)).to(torch.bfloat16).cuda()  # many ties
    u = torch.rand(20, device="cuda")
    tok, prob = ops.sample(x, u, temperature=torch.zeros(20, device="cuda"), with_prob=True)
    assert torch.equal(tok, ops.argmax(x))
    assert (prob == 1).all()
    one = ops.sample(x, u, top_k=torch.ones(20, dtype=torch.int32, device="cuda"))
    assert torch.equal(one, ops.argmax(x))
    small = ops.sample(x, u, top_p=torch.full((20,), 1e-9, device="cuda"))
    assert torch.equal(small, ops.argmax(x))


@pytest.mark.parametrize("vocab", [7, 1000, 40000])
def test_ties(ops, vocab):
    """Equal logits: every token has the same share, top-k and top-p take the lowest indices."""
    x = np.full((4, vocab), -3.0e38, np.float32)  # the lowest there is, nearly
    k = [0, 5, 0, 3]
    p = [1.0, 1.0, 0.5, 0.99]
    n = [vocab, 5, int(np.ceil(vocab * 0.5)), 3]
    want = [n_ - 1 for n_ in n]
    u = [1 - 0.4 / n_ for n_ in n]
    got, prob = run(ops, x, [1.0] * 4, k, p, [0.0] * 4, u)
    assert got.tolist() == want
    np.testing.assert_allclose(prob.cpu().numpy(), 1 / np.array(n), rtol=1e-6)


def test_ties_across_the_cut(ops):
    """A few large logits, then thousands of equal ones: top-k and top-p end inside the ties."""
    x = np.zeros((2, 30000), np.float32)
    x[:, [5, 29000, 17]] = [3.0, 4.0, 5.0]
    big = np.exp([3.0, 4.0, 5.0]).sum()
    top = [i for i in range(30000) if i not in (5, 17, 29000)]
    got, prob = run(ops, x, [1.0, 1.0], [3 + 700, 0], [1.0, (big + 999.5) / (big + 29997)], [0.0, 0.0],
                    [0.0, 0.0])
    # u = 0: the first kept token in index order; its share says how many are kept
    assert got.tolist() == [0, 0]
    np.testing.assert_allclose(prob.cpu().numpy(), [1 / (big + 700), 1 / (big + 1000)], rtol=1e-5)
    # the last tie inside the cut
    last = top[699]
    before = big - np.exp(4.0) + 699.5
    got, _ = run(ops, x[:1], [1.0], [703], [1.0], [0.0], [before / (big + 700)])
    assert got.tolist() == [last]


@pytest.mark.parametrize("vocab", [33, 9000])
def test_masked_infinite_and_nan(ops, vocab):
    x = np.random.default_rng(2).normal(0, 1, (7, vocab)).astype(np.float32)
    x[0] = -np.inf                     # nothing to draw
    x[1] = np.nan                      # nothing either
    x[2, :] = -np.inf
    x[2, 20] = -1e30                   # one token left
    x[3, ::2] = np.nan                 # NaN is masked
    x[4, 3], x[4, 30] = np.inf, np.inf  # infinite ones share the mass
    x[5] = np.finfo(np.float32).min    # the lowest value everywhere: all alike
    x[6, 4:] = np.finfo(np.float32).min
    got, prob = run(ops, x, [1.0] * 7, [0] * 7, [1.0] * 7, [0.0] * 7, [0.999999] * 7)
    got, prob = got.tolist(), prob.cpu().numpy()
    assert got[0] == got[1] == -1 and prob[0] == prob[1] == 0
    assert got[2] == 20 and prob[2] == 1
    assert got[3] % 2 == 1
    assert got[4] == 30 and prob[4] == 0.5
    assert got[5] == vocab - 1
    assert got[6] == 3
    # settings that are no numbers are off
    got, _ = run(ops, x[5:6], [1.0], [-3], [np.nan], [np.nan], [0.0])
    assert got.tolist() == [0]
    got, _ = run(ops, x[6:], [np.nan], [0], [1.0], [0.0], [0.9])
    assert got.tolist() == [int(x[6].argmax())]  # a temperature that is none is greedy


@pytest.mark.parametrize("k", [2, 300])
def test_infinite_and_signed_zero_with_top_k(ops, k):
    x = np.random.default_rng(4).normal(0, 1, (3, 9000)).astype(np.float32)
    x[0, [700, 8000, 8999]] = np.inf
    x[1] = np.where(np.arange(9000) % 2 == 0, -0.0, 0.0).astype(np.float32)  # all equal
    x[2] = -np.inf
    got, prob = run(ops, x, [1.0] * 3, [k] * 3, [1.0] * 3, [0.0] * 3, [0.99999] * 3)
    n = min(k, 3)
    assert got.tolist() == [[700, 8000, 8999][n - 1], k - 1, -1]
    np.testing.assert_allclose(prob.cpu().numpy(), [1 / n, 1 / k, 0], rtol=1e-6)
    got, _ = run(ops, x[1:2], [0.0], [0], [1.0], [0.0], [0.99999])
    assert got.tolist() == [0]


@pytest.mark.parametrize("k", [2, 50, 256, 257, 1000])
@pytest.mark.parametrize("where", ["first", "last", "one thread", "spread"])
def test_top_k_wherever_they_are(ops, k, where):
    """The k largest crowded into one slice, one thread's tokens or spread out, in falling and rising order."""
    vocab = 128256
    base = -5.0 - np.abs(np.random.default_rng(k).normal(0, 1, vocab)).astype(np.float32)
    at = {"first": np.arange(k), "last": vocab - k + np.arange(k), "one thread": 512 * 4 * np.arange(k) % vocab,
          "spread": (np.arange(k) * 7919) % vocab}[where]
    x = np.stack([base, base])
    x[0, at] = 1.0 + 0.001 * np.arange(k)
    x[1, at] = 1.0 - 0.001 * np.arange(k)
    x = x[:, :vocab]
    want = []
    for i in range(2):
        kept, _ = ref.sample_kept(x[i], 1.0, k, 1.0, 0.0)
        ids = np.flatnonzero(kept)
        assert set(ids) == set(at) or where == "one thread"
        want.append(int(ids[-1]))
    got, _ = run(ops, x, [1.0] * 2, [k] * 2, [1.0] * 2, [0.0] * 2, [0.9999999] * 2)
    assert got.tolist() == want


def test_uniform_edges(ops):
    """0, 1 and beyond, and NaN: always a kept token."""
    x = np.array([[0.0, 1.0, -np.inf, 2.0, -np.inf]] * 5, np.float32)
    got, _ = run(ops, x, [1.0] * 5, [0] * 5, [1.0] * 5, [0.0] * 5, [0.0, 1.0, 5.0, -1.0, np.nan])
    assert got.tolist() == [0, 3, 3, 0, 0]


def test_strides_offsets_and_streams(ops):
    rng = np.random.default_rng(3)
    for dtype in (torch.float32, torch.bfloat16):
        wide = torch.from_numpy(rng.normal(0, 2, (5, 3001)).astype(np.float32)).to(dtype).cuda()
        u = torch.rand(5, device="cuda")
        for lo, hi in ((0, 3001), (1, 3001), (3, 2999), (8, 2056)):
            part = wide[:, lo:hi]
            want = ops.sample(part.contiguous(), u)
            torch.cuda.synchronize()
            s = torch.cuda.Stream()
            with torch.cuda.stream(s):
                got = ops.sample(part, u)
            s.synchronize()
            assert torch.equal(got, want)


def test_frequencies(ops):
    """Evenly spread uniform numbers give every token its share, to one draw."""
    x = torch.tensor([0.0, 1.0, 2.0, -1.0, 0.5], device="cuda")
    n = 4000
    u = (torch.arange(n, device="cuda") + 0.5) / n
    got = ops.sample(x.repeat(n, 1), u)
    share = torch.bincount(got, minlength=5).double() / n
    assert (share - torch.softmax(x.double(), 0)).abs().max() <= 2.0 / n


def test_empty_and_refusals(ops):
    assert ops.sample(torch.zeros(0, 9, device="cuda"), torch.zeros(0, device="cuda")).shape == (0,)
    x, u = torch.zeros(2, 9, device="cuda"), torch.zeros(2, device="cuda")
    with pytest.raises(ValueError):
        ops.sample(x.cpu(), u)
    with pytest.raises(ValueError):
        ops.sample(x, u[:1])
    with pytest.raises(ValueError):
        ops.sample(x, u, top_k=torch.zeros(2, dtype=torch.int64, device="cuda"))
    with pytest.raises(ValueError):
        ops.sample(x.t(), u)
    with pytest.raises(ValueError):
        ops.sample(x[:1].expand(2, 9), u)
