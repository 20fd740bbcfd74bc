"""Non-finite values in batches whose thread blocks run many prompts, short ones behind long ones."""

import math

import pytest
import torch

from tests.test_serving_attention_gpu import BF16, FP16, randn
from xpu_playground_b200 import kernels as K

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,d", [(BF16, 128), (FP16, 64)])
@pytest.mark.parametrize("lens,heads", [([40] + [20] * 250, (32, 8)), ([64] * 8 + [3] * 700, (32, 8)), ([200] + [70] * 300, (4, 1)),
                                        ([20] * 40 + [40] + [20] * 400, (32, 8))])
def test_a_prompt_in_a_batch_is_the_prompt_alone(lens, heads, dtype, d):
    """Column 0 of most prompts' values is NaN or infinite: the values' other columns, and every
    other prompt, come out bit for bit as in a call of the prompt's own."""
    starts = [0]
    for n in lens:
        starts.append(starts[-1] + n)
    q, k, v = (randn(90 + i, starts[-1], h, d, dtype=dtype) for i, h in enumerate((heads[0], heads[1], heads[1])))
    for i, value in enumerate((math.nan, math.inf, 0.0, math.nan, 0.0)):
        for j in range(i, len(lens), 5):
            if value:
                v[starts[j]:starts[j + 1], :, 0] = value
    out, lse = K.prompt_attention(K.PromptPlan(lens, *heads, d), q, k, v)
    plans = {n: K.PromptPlan([n], *heads, d) for n in set(lens)}
    for a, b in zip(starts, starts[1:]):
        alone = K.prompt_attention(plans[b - a], q[a:b], k[a:b], v[a:b])
        assert torch.equal(out[a:b].view(torch.int16), alone[0].view(torch.int16)) and torch.equal(lse[a:b], alone[1])
    assert K.device_status() == 0
