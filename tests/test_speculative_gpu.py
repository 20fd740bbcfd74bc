"""Speculative decoding over the paged cache: greedy tokens as plain decoding
and the engine give them, in fewer steps; every page free in the end."""

import pytest
import torch

from xpu_playground_b200 import kernels as K
from xpu_playground_b200.qwen3 import Qwen3Engine
from xpu_playground_b200.qwen3_config import HEAD_DIM, PRESETS
from xpu_playground_b200.speculative import PagedQwen3, Server, synthetic_weights

pytestmark = pytest.mark.gpu
SHAPE, SEED, NEW = PRESETS["tiny"], 4321, 40


def prompts():
    g = torch.Generator().manual_seed(5)
    # the last one repeats itself, so that drafts are accepted
    return [torch.randint(SHAPE.vocab, (n,), generator=g).tolist() for n in (33, 1)] + [[3, 1, 4, 1, 5, 9, 2, 6] * 8]


def server(samples):
    model = PagedQwen3(SHAPE, synthetic_weights(SHAPE, SEED), 128)
    return Server(model, 3 * samples * 8, 16, 3 * samples, 128)


def assert_greedy(model, prompt, tokens, begin=0):
    """Every token from `begin` on has the largest logit of one pass over the whole text, up to
    the logit gate (2e-2, or two bf16 steps) of each of the two computations."""
    text = torch.tensor(prompt + tokens, device="cuda")
    plan = K.PromptPlan([len(text)], SHAPE.q_heads, SHAPE.kv_heads, HEAD_DIM)
    logits = model.forward(text, torch.arange(len(text), device="cuda"), lambda i, q, k, v: K.prompt_attention(plan, q, k, v)[0])
    at = torch.arange(len(prompt) - 1 + begin, len(text) - 1, device="cuda")
    top = logits[at].float().max(-1).values
    gate = torch.maximum(torch.full_like(top, 2e-2), 2 * 2.0 ** (torch.floor(torch.log2(top.abs())) - 7))
    assert bool((logits[at, text[at + 1]].float() >= top - 2 * gate).all())


@pytest.mark.parametrize("width", [0, 4])
def test_tokens_are_greedy_and_pages_come_back(width):
    s = server(2)
    got = s.generate(prompts(), NEW, samples=2, width=width, depth=6)
    for prompt, samples in zip(prompts(), got):
        assert [len(t) for t in samples] == [NEW, NEW] and samples[0][0] != samples[1][0]
        for i, tokens in enumerate(samples):
            assert_greedy(s.model, prompt, tokens, begin=i)  # sample 1 begins with the second best
    assert s.steps == NEW - 1 if width == 0 else s.steps <= NEW - 1
    assert s.emitted >= 6 * (NEW - 1)
    assert int(s.cache.refs.sum()) == 0 and int(s.cache.lens.sum()) == 0 and bool((s.cache.tables == -1).all())


def test_tokens_are_the_engines():
    engine = Qwen3Engine(SHAPE, 128)
    engine.init_synthetic(SEED)
    s = server(1)
    for prompt, (tokens,) in zip(prompts(), s.generate(prompts(), NEW, samples=1, width=3, depth=4)):
        want = engine.generate(prompt, NEW)
        assert_greedy(s.model, prompt, tokens)
        assert_greedy(s.model, prompt, want)  # the engine's tokens by the example's logits
    engine.close()


def test_command():
    from xpu_playground_b200.speculative import main
    assert main(["--new-tokens", "6", "--prompts", "2", "--prompt-len", "20", "--samples", "1"]) == 0
