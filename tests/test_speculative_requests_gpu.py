"""Several requests to one server of the speculative example: each is drawn with random numbers of its own."""

import pytest
import torch

from tests.test_speculative_gpu import prompts
from tests.test_speculative_sampling_gpu import server
from xpu_playground_b200.speculative import Sampling

pytestmark = pytest.mark.gpu


def requests(width, samples=2):
    """Tokens and random numbers of three requests in turn, the last one with fewer prompts."""
    s, got = server(samples, Sampling(1.0, seed=1)), []
    for given in (prompts(), prompts(), prompts()[:2]):
        tokens = s.generate(given, 12, samples=samples, width=width)
        got.append((tokens, s.u.clone()))
    return got


def test_the_same_prompt_is_drawn_anew():
    (a, u), (b, v), (c, w) = requests(0)
    for x, y in zip(a, b):
        assert x[0] != y[0] and x[1] != y[1]
    assert a[:2] != c and b[:2] != c
    assert float((u == v).float().mean()) < 1e-3  # 24 bits each: two alike by chance are rare
    used, left = [0, 1, 2, 3], [4, 5]  # two prompts of two samples; the other places keep theirs
    assert float((v[used] == w[used]).float().mean()) < 1e-3 and torch.equal(v[left], w[left])


def test_the_seed_and_the_requests_before_decide():
    first, again, drafted = requests(0), requests(0), requests(4)
    for (a, u), (b, v), (_, w) in zip(first, again, drafted):
        assert a == b and torch.equal(u, v) and torch.equal(u, w)  # drafts use up no numbers


def test_greedy_requests_repeat():
    s = server(2)
    assert s.generate(prompts(), 12, samples=2, width=0) == s.generate(prompts(), 12, samples=2, width=0)
