"""Products of many 8-bit rows, which pairs of blocks compute in tiles of 256 x 256 (k_wide in fp8_gemm.cu)."""

import pytest
import torch

from tests._fp8 import check_product, product
from tests._graphs import kernels_of
from tests.test_fp8_chain_gpu import Layer, settings
from tests.test_fp8_gemm_gpu import BF16, FP16, operands
from xpu_playground_b200 import kernels as K

pytestmark = pytest.mark.gpu


def by_pairs(*args, **kwargs):
    names = kernels_of(lambda: K.fp8_gemm(*args, **kwargs))
    assert len(names) == 1 and ("k_wide" in names[0]) != ("k_skinny" in names[0]), names
    return "k_wide" in names[0]


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("m,n,k", [(4100, 2056, 1040), (2049, 1999, 1168)])
def test_scales_that_jump_from_group_to_group(m, n, k, dtype):
    """Scales of a group go from one warp to others four groups at a time: those of another group, or of the tile before, would
    be off by a factor of 64 at least. Each pair has one to three tiles of 9 or 10 groups, so that places are used over and over."""
    a, a_scales, w, w_scales = operands(m, n, k, m, 0.0)
    blocks = len(a_scales)
    jump = 8.0 ** torch.tensor([[0, 3, 1, 4, 2][g % 5] for g in range(blocks)], device="cuda")  # neighbours differ
    a_scales *= jump[:, None] * 1e-4 * (1 + torch.arange(m, device="cuda") % 7)
    w_scales *= jump.flip(0)[None, :] * (1 + torch.arange(len(w_scales), device="cuda") % 3)[:, None]
    if dtype == FP16:
        w_scales *= 1e-2
    assert by_pairs(a, a_scales, w, w_scales, dtype=dtype)
    first = K.fp8_gemm(a, a_scales, w, w_scales, dtype=dtype)
    check_product(first, *product(a, a_scales, w, w_scales), k)
    again = torch.empty_like(first)
    for i in range(200):
        if i % 5 == 0:
            K.fp8_quantize(first[:64, :1920].contiguous())  # another kernel before it now and then
        K.fp8_gemm(a, a_scales, w, w_scales, out=again)
        assert torch.equal(again, first)
    assert K.device_status() == 0


def test_calls_of_one_group_one_after_the_other():
    """A pair ends as soon as its only group is done, and another block takes its place: both blocks stay until every arrival of
    the products on their barriers is in."""
    calls = [operands(m, n, k, i, 1.0) for i, (m, n, k) in enumerate([(257, 9999, 16), (777, 4096, 128), (300, 7000, 112), (20, 640, 128)])]
    assert [by_pairs(*x) for x in calls] == [True, True, True, False]
    want = [K.fp8_gemm(*x) for x in calls]
    for x, c in zip(calls, want):
        check_product(c, *product(*x), x[0].shape[1])
    outs = [[torch.empty_like(c) for c in want] for _ in range(8)]
    for _ in range(25):
        for out in outs:
            for x, c in zip(calls, out):
                K.fp8_gemm(*x, out=c)
    torch.cuda.synchronize()
    assert all(torch.equal(c, w) for out in outs for c, w in zip(out, want))
    assert K.device_status() == 0


# n on both sides of a multiple of 8 (whole rows leave by a copy of tiles, others value by value), of 64 and of 256; half a tile
# behind the last whole one (n % 256 <= 128); m one row behind a tile; 1 to 10 groups, the last one short; up to three tiles a pair.
PAIRS = [(777, 4096, 272), (1025, 3001, 144), (2049, 1999, 400), (257, 9999, 16), (4100, 2056, 1040), (600, 4224, 512), (700, 4000, 640),
         (1300, 8200, 768), (512, 4608, 896), (300, 7001, 1024), (2300, 3330, 1168), (1793, 4161, 128), (70, 24000, 256), (9000, 257, 256)]
ROWS = [(128, 4096, 512), (300, 4096, 256), (2048, 640, 512), (65, 11000, 128), (777, 384, 1536)]


@pytest.mark.parametrize("m,n,k,pairs", [(*s, True) for s in PAIRS] + [(*s, False) for s in ROWS])
@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_product(m, n, k, pairs, dtype):
    a, a_scales, w, w_scales = operands(m, n, k, m + n + k, 3.0 if dtype == BF16 else 1.0)  # inside fp16's range
    if dtype == FP16:
        w_scales *= 1e-2
    assert by_pairs(a, a_scales, w, w_scales, dtype=dtype) == pairs
    check_product(K.fp8_gemm(a, a_scales, w, w_scales, dtype=dtype), *product(a, a_scales, w, w_scales), k)


@pytest.mark.parametrize("n", [6000, 5999])
def test_a_bad_row_stays_alone(n):
    """NaN and infinite scales reach their own row, or their own 128 columns, and no other: in either block, in the first and the last
    tile."""
    m, k = 1100, 400
    a, a_scales, w, w_scales = operands(m, n, k, 3, 0.0)
    assert by_pairs(a, a_scales, w, w_scales)
    want = K.fp8_gemm(a, a_scales, w, w_scales)
    a_scales[1, 5], a_scales[3, 200], a_scales[0, 1099] = float("nan"), float("inf"), float("nan")
    a.view(torch.uint8)[131, 17] = 0x7F
    a.view(torch.uint8)[1024, 399] = 0xFF
    w.view(torch.uint8)[1000, 0] = 0x7F
    w_scales[2, 3], w_scales[-1, 0] = float("inf"), float("nan")
    got = K.fp8_gemm(a, a_scales, w, w_scales)
    bad = torch.zeros(m, n, dtype=torch.bool, device="cuda")
    bad[[5, 200, 1099, 131, 1024]] = True
    bad[:, 256:384] = bad[:, 1000] = bad[:, (n - 1) // 128 * 128:] = True
    assert not torch.isfinite(got[bad]).any() and torch.equal(got[~bad], want[~bad])


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("m,n,k", [(513, 8192, 512), (1025, 4099, 400), (4100, 2056, 1040)])
def test_products_repeat_and_memory_behind_them_stays(m, n, k, dtype):
    args = operands(m, n, k, 5, 1.0)
    args[3].mul_(1e-2)
    held = torch.full((m * n + 4096,), 7.0, dtype=dtype, device="cuda")
    out = held[:m * n].view(m, n)
    assert by_pairs(*args, out=out)
    assert K.fp8_gemm(*args, out=out) is out
    for _ in range(5):
        assert torch.equal(K.fp8_gemm(*args, dtype=dtype), out)
    assert (held[m * n:] == 7).all()


def test_scales_and_operands_behind_the_last_row_are_not_read_as_values():
    """Rows behind the last tile row's end and blocks behind n hold NaN in the memory that follows."""
    m, n, k = 777, 4000, 272
    a, a_scales, w, w_scales = operands(m, n, k, 9, 1.0)
    want = K.fp8_gemm(a, a_scales, w, w_scales)

    def followed(t):
        bytes_ = t.contiguous().view(torch.uint8).flatten()
        held = torch.full((bytes_.numel() + (1 << 20),), 0xFF, dtype=torch.uint8, device="cuda")  # NaN of either type
        held[:bytes_.numel()] = bytes_
        return held[:bytes_.numel()].view(t.dtype).view(t.shape)

    args = [followed(t) for t in (a, a_scales, w, w_scales)]
    assert by_pairs(*args) and torch.equal(K.fp8_gemm(*args), want)


@pytest.mark.parametrize("n", [16400, 16391])
def test_outputs_past_32_bits(n):
    """Rows whose place in c is past 2^31 elements."""
    m, k = 131_100, 16
    a, a_scales, w, w_scales = operands(m, n, k, 7, 1.0)
    c = K.fp8_gemm(a, a_scales, w, w_scales)
    assert c.numel() > 1 << 31
    for rows in (slice(0, 300), slice(65_500, 65_600), slice(m - 700, m)):
        part = a[rows], a_scales[:, rows].contiguous(), w, w_scales
        check_product(c[rows], *product(*part), k)


@pytest.mark.parametrize("rows", [400, 1000])
def test_a_layer_and_its_answer(rows):
    """A layer whose largest products go to pairs of blocks: in a row, captured and replayed, between products of 16-bit rows."""
    layer, choice = Layer(BF16, 5), settings(rows)
    given = layer.inputs(rows)
    names = kernels_of(lambda: layer.run(*given, choice))
    assert any("k_wide" in n for n in names) and any("k_skinny" in n for n in names)
    want = layer.run(*given, choice)
    layer.check(*given, choice, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = layer.run(*given, choice)
    for _ in range(5):
        graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(p.float(), q.float()) for p, q in zip(want, got))
    x, w = torch.randn(300, 512, device="cuda").bfloat16(), torch.randn(640, 512, device="cuda").bfloat16()
    other = K.gemm_bt(x, w)
    for _ in range(10):
        y = K.gemm_bt(x, w)
        got = layer.run(*given, choice)
        z = K.gemm_bt(x, w)
        assert torch.equal(y, other) and torch.equal(z, other)
        assert all(torch.equal(p.float(), q.float()) for p, q in zip(want, got))
    assert K.device_status() == 0


def test_on_two_streams_at_once():
    """Each call has its own outputs and no workspace: any number may be under way."""
    calls = [operands(m, n, k, i, 1.0) for i, (m, n, k) in enumerate([(1025, 4099, 400), (700, 4000, 640), (40, 6144, 1024)])]
    want = [K.fp8_gemm(*x) for x in calls]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in calls]
    got = [[K.fp8_gemm(*x, stream=s) for _ in range(20)] for x, s in zip(calls, streams)]
    torch.cuda.synchronize()
    assert all(torch.equal(c, w) for outs, w in zip(got, want) for c in outs)
    assert K.device_status() == 0
