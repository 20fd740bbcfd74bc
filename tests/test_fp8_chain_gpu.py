"""The 8-bit operators and sampling as a decoder layer and its answer use them: one after the other without a wait, captured and
replayed, on another stream; each result checked against its definition from the inputs that it had."""

import pytest
import torch

from tests._fp8 import check_product, check_rows, choose, product
from tests.test_fp8_rows_gpu import NORM_OFF, norm64, silu
from xpu_playground_b200 import kernels as K
from xpu_playground_b200.fp8 import Fp8Weight

pytestmark = pytest.mark.gpu
HIDDEN, INNER, VOCABULARY = 512, 1040, 4099
BF16, FP16 = torch.bfloat16, torch.float16


class Layer:
    def __init__(self, dtype, seed=0):
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.dtype = dtype
        self.w = {n: Fp8Weight(torch.randn(*s, device="cuda", generator=g) * 0.05) for n, s in
                  dict(out=(HIDDEN, HIDDEN), gate_up=(2 * INNER, HIDDEN), down=(HIDDEN, INNER), head=(VOCABULARY, HIDDEN)).items()}
        self.norms = [(1 + 0.1 * torch.randn(HIDDEN, device="cuda", generator=g)).to(dtype) for _ in range(2)]
        self.g = g

    def inputs(self, rows):
        attention, residual = (torch.randn(rows, HIDDEN, device="cuda", generator=self.g).to(self.dtype) for _ in range(2))
        return attention, residual, torch.rand(rows, device="cuda", generator=self.g)

    def run(self, attention, residual, u, settings, stream=None):
        """Everything that is made, in order."""
        s = dict(stream=stream)
        a = K.fp8_quantize(attention, **s)
        x = self.w["out"](a, self.dtype, **s)
        first = K.fp8_rms_norm(x, self.norms[0], residual, 1e-6, **s)
        gate_up = self.w["gate_up"](first[1:], self.dtype, **s)
        h = K.fp8_silu_multiply(gate_up, **s)
        y = self.w["down"](h, self.dtype, **s)
        last = K.fp8_rms_norm(y, self.norms[1], first[0], 1e-6, **s)
        logits = self.w["head"](last[1:], self.dtype, **s)
        return [*a, x, *first, gate_up, *h, y, *last, logits, *K.sample(logits, u, *settings, **s)]

    def check(self, attention, residual, u, settings, got):
        qa, sa, x, t1, q1, s1, gate_up, qh, sh, y, t2, q2, s2, logits, tokens, logprobs = got
        check_rows(qa, sa, attention.double().cpu(), 0.0)
        for q, s, name, c in ((qa, sa, "out", x), (q1, s1, "gate_up", gate_up), (qh, sh, "down", y), (q2, s2, "head", logits)):
            want, size = product(q, s, self.w[name].q, self.w[name].scales)
            check_product(c, want, size, q.shape[1])
        for a, b, t, q, s, norm in ((x, residual, t1, q1, s1, self.norms[0]), (y, t1, t2, q2, s2, self.norms[1])):
            assert torch.equal(t, (a.float() + b.float()).to(self.dtype))
            check_rows(q, s, norm64(t.cpu(), norm.cpu(), 1e-6), NORM_OFF)
        gate, up = gate_up.double().cpu().chunk(2, 1)
        check_rows(qh, sh, silu(gate) * up, 2.0 ** -16)
        names = ("temperature", "top_k", "top_p", "min_p")
        for i in range(len(u)):
            token, logprob = choose(logits[i].double().cpu().numpy(), float(u[i]), **{n: v[i].item() for n, v in zip(names, settings)})
            assert int(tokens[i]) == token and abs(float(logprobs[i]) - logprob) <= 2.0 ** -24 * abs(logprob) + 1e-10


def settings(rows):
    pick = lambda values, dtype: torch.tensor([values[i % len(values)] for i in range(rows)], dtype=dtype, device="cuda")  # noqa: E731
    return (pick([1.0, 0.0, 0.7, 1.3, 0.5], torch.float32), pick([0, 5, 40, 0, 300, 0, 1], torch.int32),
            pick([1.0, 0.9, 0.5], torch.float32), pick([0.0, 0.05], torch.float32))


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("rows", [1, 7, 64, 65, 300])
def test_a_layer_and_its_answer(rows, dtype):
    layer, choice = Layer(dtype), settings(rows)
    given = layer.inputs(rows)
    layer.check(*given, choice, layer.run(*given, choice))


@pytest.mark.parametrize("rows", [1, 33, 300])
def test_captured_and_replayed(rows):
    """Twice from one graph, with new inputs in the same place, and beside a second graph of the same layer."""
    layer, choice = Layer(BF16, 1), settings(rows)
    graphs = []
    for _ in range(2):
        given = layer.inputs(rows)
        want = layer.run(*given, choice)  # warms up
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = layer.run(*given, choice)
        graphs.append((graph, given, want, got))
    for _ in range(3):
        for graph, *_ in graphs:
            graph.replay()
    torch.cuda.synchronize()
    for _, _, want, got in graphs:
        assert all(torch.equal(a.float(), b.float()) for a, b in zip(want, got))
    graph, given, _, got = graphs[0]
    for old, new in zip(given, layer.inputs(rows)):
        old.copy_(new)
    graph.replay()
    torch.cuda.synchronize()
    layer.check(*given, choice, got)


def test_two_graphs_at_once():
    layer, choice = Layer(BF16, 2), settings(40)
    runs = []
    for _ in range(2):
        given = layer.inputs(40)
        want = layer.run(*given, choice)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = layer.run(*given, choice)
        runs.append((graph, torch.cuda.Stream(), want, got, given))  # a graph's inputs stay where they are
    torch.cuda.synchronize()
    for _ in range(20):
        for graph, stream, *_ in runs:
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize()
    for _, _, want, got, _ in runs:
        assert all(torch.equal(a.float(), b.float()) for a, b in zip(want, got))


@pytest.mark.parametrize("rows", [3, 200])
def test_on_a_given_stream(rows):
    """Inputs that are still on their way there: the calls queue behind them, and their outputs are that stream's memory."""
    layer, choice, side = Layer(BF16, 3), settings(rows), torch.cuda.Stream()
    given, later = layer.inputs(rows), layer.inputs(rows)
    want = layer.run(*later, choice)
    side.wait_stream(torch.cuda.current_stream())
    held = torch.full((1 << 22,), 7.0, device="cuda")
    torch.cuda.synchronize()
    torch.cuda._sleep(20_000_000)
    copy = held.clone()
    del held  # free for the current stream's next allocation, and for no other's
    with torch.cuda.stream(side):
        torch.cuda._sleep(5_000_000)
        for old, new in zip(given, later):
            old.copy_(new)
    got = layer.run(*given, choice, stream=side)
    torch.cuda.synchronize()
    assert bool((copy == 7).all()) and all(torch.equal(a.float(), b.float()) for a, b in zip(want, got))


def test_other_operators_around_them():
    """Products of both kinds one after the other: none starts before the one before it has let go of its TMEM."""
    layer, choice = Layer(BF16, 4), settings(70)
    given = layer.inputs(70)
    want = layer.run(*given, choice)
    a, w = torch.randn(300, 512, device="cuda").bfloat16(), torch.randn(640, 512, device="cuda").bfloat16()
    other = K.gemm_bt(a, w)
    for _ in range(10):
        x = K.gemm_bt(a, w)
        got = layer.run(*given, choice)
        y = K.gemm_bt(a, w)
        assert torch.equal(x, other) and torch.equal(y, other)
        assert all(torch.equal(p.float(), q.float()) for p, q in zip(want, got))
    assert K.device_status() == 0
