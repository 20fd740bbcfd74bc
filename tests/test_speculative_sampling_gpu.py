"""Drawn tokens and 8-bit projections in the speculative example."""

import numpy as np
import pytest
import torch

from tests.test_speculative_gpu import NEW, SEED, SHAPE, prompts
from xpu_playground_b200 import kernels as K
from xpu_playground_b200.qwen3_config import HEAD_DIM
from xpu_playground_b200.speculative import PagedQwen3, Sampling, Server, synthetic_weights

pytestmark = pytest.mark.gpu


def model(eight_bits=False):
    return PagedQwen3(SHAPE, synthetic_weights(SHAPE, SEED), 128, eight_bits)


def server(samples, sampling=None, eight_bits=False):
    return Server(model(eight_bits), 3 * samples * 8, 16, 3 * samples, 128, sampling)


def all_logits(m, text):
    plan = K.PromptPlan([len(text)], SHAPE.q_heads, SHAPE.kv_heads, HEAD_DIM)
    return m.forward(torch.tensor(text, device="cuda"), torch.arange(len(text), device="cuda"),
                     lambda i, q, k, v: K.prompt_attention(plan, q, k, v)[0])


@pytest.mark.parametrize("eight_bits", [False, True])
@pytest.mark.parametrize("choice", [Sampling(0.0), Sampling(0.7, top_k=1)])
def test_no_choice_is_the_greedy_token(choice, eight_bits):
    a = server(1, None, eight_bits).generate(prompts(), NEW, width=0)
    assert server(1, choice, eight_bits).generate(prompts(), NEW, width=0) == a


@pytest.mark.parametrize("width", [0, 4])
@pytest.mark.parametrize("choice", [Sampling(1.0, seed=3), Sampling(0.8, 50, 0.9, 0.02, seed=4)])
def test_drawn_tokens_are_where_their_random_numbers_fall(choice, width):
    """Each token's share of the kept weights, by one pass over the whole text, holds its random number, up to what two
    computations' logits differ by (2e-2 each, as for greedy tokens): weights by a factor of exp(4e-2 / temperature), sums
    of them by as much, twice for a quotient; top-k, top-p and min-p take logits within that distance of their border too."""
    s = server(2, choice)
    for p, (prompt, samples) in enumerate(zip(prompts(), s.generate(prompts(), NEW, samples=2, width=width))):
        assert samples[0] != samples[1]
        for i, tokens in enumerate(samples):
            slot = p if i == 0 else 3 + p
            logits = all_logits(s.model, prompt + tokens).double().cpu().numpy()
            for at, token in enumerate(tokens):
                x = logits[len(prompt) - 1 + at]
                u, slack = float(s.u[slot, len(prompt) - 1 + at]), 0.04
                gate = np.expm1(2 * slack / choice.temperature)
                larger, as_large = x > x[token] + slack, x >= x[token] - slack
                w = np.exp((x - x.max()) / choice.temperature)
                if choice.top_k:
                    assert larger.sum() < choice.top_k
                top = np.sort(w)[::-1][:choice.top_k or None]
                assert w[larger].sum() < choice.top_p * top.sum() * (1 + gate) and w[token] >= choice.min_p * (1 - gate)
                kept = top[np.concatenate([[0], np.cumsum(top)[:-1]]) < choice.top_p * top.sum()]
                kept = kept[kept >= choice.min_p]
                low, high = w[larger].sum() / kept.sum() * (1 - gate), w[as_large].sum() / kept.sum() * (1 + gate)
                # a token more or less at the end of what is kept
                assert low - 2 * gate <= u <= high + 2 * gate
    assert int(s.cache.refs.sum()) == 0


def test_the_seed_decides():
    a, b, c = (server(2, Sampling(1.0, seed=i)).generate(prompts(), 12, samples=2, width=0) for i in (1, 1, 2))
    assert a == b and a != c


def test_eight_bits_are_near_sixteen():
    """A product of two operands rounded to e4m3 is off by 2^-4 / sqrt(3) of its terms each, 5% in all; the stream of two layers
    takes four such products, one after the other, before the last one: sqrt(5) x 5% and some for the 8-bit
    rounding of what the nonlinear parts get. Twice that is the bound."""
    text = prompts()[0]
    a, b = all_logits(model(), text).double(), all_logits(model(True), text).double()
    assert float((a - b).norm() / a.norm()) < 0.25


def test_eight_bits_serve():
    s = server(2, None, True)
    got = s.generate(prompts(), NEW, samples=2, width=4)
    assert [[len(t) for t in x] for x in got] == [[NEW, NEW]] * 3 and s.emitted >= 6 * (NEW - 1)
    assert int(s.cache.refs.sum()) == 0 and s.cache.status() == 0 and K.device_status() == 0


def test_command():
    from xpu_playground_b200.speculative import main
    assert main(["--new-tokens", "6", "--prompts", "2", "--prompt-len", "20", "--samples", "2", "--eight-bits", "--temperature", "0.7",
                 "--top-k", "20", "--top-p", "0.95", "--min-p", "0.01"]) == 0
