"""examples/paged_generate.py: the 4-bit cache, its attention and the sampler in one decoder."""
import importlib.util
from pathlib import Path

import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def example(built_lib):
    path = Path(__file__).resolve().parent.parent / "examples" / "paged_generate.py"
    spec = importlib.util.spec_from_file_location("paged_generate", path)
    m = importlib.util.module_from_spec(spec)
    import sys
    sys.modules["paged_generate"] = m
    spec.loader.exec_module(m)
    return m


def prompts(vocab, lengths):
    g = torch.Generator().manual_seed(1)
    return [torch.randint(0, vocab, (n,), generator=g).tolist() for n in lengths]


def test_generates_and_repeats(example):
    model = example.Decoder(example.Config(layers=2))
    asked = prompts(model.c.vocab, (5, 33, 1, 61))
    a = example.generate(model, asked, 20, seed=3)
    assert a.shape == (4, 20) and (a >= 0).all() and (a < model.c.vocab).all()
    assert torch.equal(a, example.generate(model, asked, 20, seed=3))
    assert not torch.equal(a, example.generate(model, asked, 20, seed=4))


def test_prompt_at_once_or_token_by_token(example):
    """The logits after a prompt do not hang on how it was fed, to the rounding of bf16 activations:
    every layer's inputs are rounded to 2^-9, two layers and the head add up to a few of them."""
    c = example.Config(layers=2)
    model = example.Decoder(c)
    prompt = torch.tensor(prompts(c.vocab, (37,))[0], device="cuda")

    def i32(a):
        return torch.tensor(a, dtype=torch.int32, device="cuda")

    whole = model.logits(prompt, i32([[4, 2, 9]]), i32([0, 37]), i32([37])).double()
    for y in model.layers:
        y.cache = example.ops.kv4_cache(c.num_pages, c.page_size, c.n_kv, c.head_dim)
    for i in range(37):
        last = model.logits(prompt[i:i + 1], i32([[1, 0, 5]]), i32([0, 1]), i32([i + 1])).double()
    # a code of the cache may also flip by one step: 0.1 of the logits' spread leaves room for both
    assert (whole - last).norm() <= 0.1 * whole.norm()
